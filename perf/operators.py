"""What is measured of the speculative-decoding operators.

A serving program that verifies drafted tokens makes five calls a step and layer:

  plan       block tables, slot maps, positions and tree masks of a batch, built on the GPU from its lengths
  rope       RMS norm of every query and key head and the position rotation in one pass, the keys and values
             written into their pool slots on the way where the caller asks for it
  rope_grad  the gradients of that pass (training)
  tree       attention of a tree of drafted tokens over a paged cache (f32, f16 or e4m3 pools)
  commit     the accepted path's keys and values moved to the end of the sequence

A case is a dict of plain values.  ``prepare`` makes what the program holds before the call, ``run`` makes one pass:
the plain form in 32 bits with elementary torch operations, or, where ``own`` is true, the framework's call.  ``exact``
is the definition in 64 bits.  Lengths and the drafted trees' shapes come from the case's ``draw``; values, block
numbers and accepted paths come from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F32, F16, E4M3 = 0, 1, 2
TORCH = {F32: torch.float32, F16: torch.float16, E4M3: torch.uint8}
ELEM = {F32: 4, F16: 2, E4M3: 1}
IO = {F32: 4, F16: 2, E4M3: 2}
BASE, EPS = 10000.0, 1e-6

# (query heads, kv heads): the benchmark's and the test sweeps' head layouts
HEADS = [(8, 8), (16, 4), (32, 8), (64, 8), (16, 16), (32, 32), (8, 1), (12, 4), (32, 2)]


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # a handful of chats decoding one token each: the smallest plan, launch latency alone
        dict(name="plan_b8", kind="plan", batch=8, ctx_lo=128, ctx_hi=4096, nodes_lo=1, nodes_hi=1, block=16, tree=False,
             draw=1),
        # a large batch with a long tail of lengths, a drafted tree for every request
        dict(name="plan_b256_tree", kind="plan", batch=256, ctx_lo=16, ctx_hi=8192, nodes_lo=8, nodes_hi=64, block=16,
             tree=True, draw=2),
        # a decode batch of 64 tokens straight into the f16 pools
        dict(name="rope_f16_decode", kind="rope", dtype=F16, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             tokens=64, pos_lo=128, pos_hi=4096, append=True, block=16, draw=3),
        # a long prompt's projections, half of each f32 head rotated, far positions, an odd count of tokens
        dict(name="rope_f32_prompt", kind="rope", dtype=F32, heads=16, kv_heads=4, dim=128, rotary=64, interleaved=True,
             tokens=4133, pos_lo=100000, pos_hi=131072, append=False, block=16, draw=4),
        # training: 8 K tokens of the f16 grouped-query layer
        dict(name="rope_grad_f16", kind="rope_grad", dtype=F16, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, tokens=8192, pos_lo=0, pos_hi=8192, draw=5),
        # training in f32 at head size 64, a short ragged batch
        dict(name="rope_grad_f32", kind="rope_grad", dtype=F32, heads=8, kv_heads=2, dim=64, rotary=64, interleaved=True,
             tokens=600, pos_lo=0, pos_hi=2048, draw=6),
        # one interactive user: 8 drafted tokens over 4 K of context
        dict(name="tree_f16_b1", kind="tree", dtype=F16, heads=32, kv_heads=8, dim=128, block=16, batch=1, ctx_lo=4133,
             ctx_hi=4133, nodes_lo=8, nodes_hi=8, window=0, draw=7),
        # a serving batch, up to 64 drafted tokens a request: bytes and matrix work about equal
        dict(name="tree_f16_b16", kind="tree", dtype=F16, heads=32, kv_heads=8, dim=128, block=16, batch=16, ctx_lo=128,
             ctx_hi=4096, nodes_lo=16, nodes_hi=64, window=0, draw=8),
        # long contexts over quantised pools, 64 query heads: the largest
        dict(name="tree_e4m3_long", kind="tree", dtype=E4M3, heads=64, kv_heads=8, dim=128, block=16, batch=4,
             ctx_lo=16384, ctx_hi=65536, nodes_lo=32, nodes_hi=32, window=0, draw=9),
        # an f32 layer of head size 64, blocks of 8, odd trees
        dict(name="tree_f32_odd", kind="tree", dtype=F32, heads=8, kv_heads=2, dim=64, block=8, batch=6, ctx_lo=3,
             ctx_hi=1000, nodes_lo=5, nodes_hi=13, window=0, draw=10),
        # a small batch's accepted paths
        dict(name="commit_f16_b16", kind="commit", dtype=F16, kv_heads=8, dim=128, block=16, batch=16, ctx_lo=128,
             ctx_hi=1024, nodes_lo=16, nodes_hi=64, draw=11),
        # a large batch over f32 pools, wide trees
        dict(name="commit_f32_b128", kind="commit", dtype=F32, kv_heads=8, dim=128, block=16, batch=128, ctx_lo=16,
             ctx_hi=256, nodes_lo=32, nodes_hi=128, draw=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(["plan", "rope", "rope", "rope_grad", "rope_grad", "tree", "tree", "tree", "tree", "commit"])
    heads, kv = rng.choice(HEADS)
    c = dict(kind=kind, block=rng.choice([16, 16, 8, 32, 64]), draw=rng.randrange(1 << 20))
    if kind in ("rope", "rope_grad"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        lo = _log_int(rng, 1, 1 << 20) - 1
        c.update(dtype=rng.choice([F32, F16]), heads=heads, kv_heads=kv, dim=dim, rotary=rng.choice([dim, dim, dim // 2]),
                 interleaved=rng.random() < 0.5, tokens=_log_int(rng, 1, 8192), pos_lo=lo,
                 pos_hi=lo + _log_int(rng, 1, 8192))
        if kind == "rope":
            c["append"] = rng.random() < 0.5
        return c
    hi = _log_int(rng, 16, 32768)
    nodes = _log_int(rng, 1, 128)
    c.update(batch=_log_int(rng, 1, 256), ctx_lo=rng.randint(0, max(1, hi // 4)), ctx_hi=hi,
             nodes_lo=rng.randint(1, nodes), nodes_hi=nodes)
    if kind == "plan":
        c["tree"] = rng.random() < 0.5
    elif kind == "tree":
        c.update(dtype=rng.choice([F32, F16, F16, E4M3, E4M3]), heads=heads, kv_heads=kv,
                 dim=rng.choice([64, 80, 96, 128, 128, 128, 256]), window=rng.choice([0, 0, rng.randint(1, 4096)]))
    else:
        c.update(dtype=rng.choice([F32, F16]), kv_heads=kv, dim=rng.choice([64, 80, 128, 256]))
    return c


def draw(rng):
    while True:
        c = _draw_once(rng)
        w = work(c)
        if c["kind"] in ("rope", "rope_grad"):
            ok = w["bytes"] <= 2.6e8
        elif c["kind"] == "plan":
            ok = True
        elif c["kind"] == "commit":
            ok = c["batch"] * (c["ctx_hi"] + 128) * c["kv_heads"] * c["dim"] <= 1e8
        else:  # the plain form holds the padded keys and scores in 32 bits
            long = c["ctx_hi"] + c["nodes_hi"]
            ok = (c["batch"] * long * c["kv_heads"] * c["dim"] <= 3e8 and
                  c["batch"] * long * c["nodes_hi"] * c["heads"] <= 4e8 and
                  w["flops"] <= (8e10 if c["dim"] == 128 and c["dtype"] != F32 else 1e10))
        if ok:
            return c


# ------------------------------------------------------------------ sizes


def _shape(c):
    """Cached tokens and drafted tokens of every sequence, and the drafted tokens' parents [batch, nodes] (-1: the
    cached context; a node's parent comes before it), fixed by the case."""
    r = np.random.default_rng(c["draw"])
    n = c["batch"]
    ctx = r.integers(c["ctx_lo"], c["ctx_hi"] + 1, n)
    if c["ctx_hi"] >= 64 * max(1, c["ctx_lo"]):  # a long tail
        x = np.exp(r.normal(math.log(math.sqrt(max(1, c["ctx_lo"]) * c["ctx_hi"])), 1.0, n))
        ctx = np.clip(np.round(x), c["ctx_lo"], c["ctx_hi"])
    new = r.integers(c["nodes_lo"], c["nodes_hi"] + 1, n)
    i = np.arange(c["nodes_hi"])[None, :]
    parents = np.floor(i * r.random((n, c["nodes_hi"])) ** 0.5).astype(np.int64)
    parents[:, 0] = -1
    return ctx.astype(np.int64), new.astype(np.int64), parents


def _seen(c):
    """Drafted tokens on every node's path, itself among them."""
    ctx, new, parents = _shape(c)
    depth = np.ones(parents.shape, np.int64)
    for i in range(1, parents.shape[1]):
        depth[:, i] = 1 + depth[np.arange(len(new)), parents[:, i]]
    return depth


def work(c):
    kind = c["kind"]
    if kind in ("rope", "rope_grad"):
        e, n = IO[c["dtype"]], c["tokens"]
        x = n * (c["heads"] + c["kv_heads"]) * c["dim"]
        b = (2 if kind == "rope" else 3) * x * e + 4 * n
        if kind == "rope" and c["append"]:
            b += 2 * n * c["kv_heads"] * c["dim"] * e + 8 * n
        return {"bytes": float(b), "flops": float((8 if kind == "rope" else 20) * x)}
    ctx, new, _ = _shape(c)
    rows = int(new.sum())
    if kind == "plan":
        blocks = int(((ctx + new + c["block"] - 1) // c["block"]).sum())
        width = int(((ctx + new + c["block"] - 1) // c["block"]).max())
        b = 8 * len(ctx) + 4 * blocks + 8 * len(ctx) + 4 * len(ctx) * width + rows * (4 + 8)
        b += rows * (4 + 8 * _words(c)) if c["tree"] else 0
        return {"bytes": float(b), "flops": float(rows)}
    tok = 2 * c["kv_heads"] * c["dim"] * ELEM[c["dtype"]]
    if kind == "commit":  # the first node's token is where it belongs
        n = sum(len(p) - 1 for p in _paths(c, 0))
        return {"bytes": float(2 * n * tok + 4 * len(ctx) * 10), "flops": float(max(1, n))}
    seen = _seen(c)
    live = np.arange(c["nodes_hi"])[None, :] < new[:, None]
    keys = ctx[:, None] + seen
    span = ctx + new
    if c["window"]:
        keys = np.minimum(keys, c["window"])
        span = np.minimum(span, c["window"] + new)
    pairs = int((keys * live).sum())
    b = int(span.sum()) * tok + 2 * rows * c["heads"] * c["dim"] * IO[c["dtype"]] + rows * 8 * _words(c)
    if c["dtype"] == E4M3:
        b += int(span.sum()) // c["block"] * 4
    return {"bytes": float(b), "flops": float(4 * c["dim"] * c["heads"] * pairs)}


def _words(c):
    return (c["nodes_hi"] + 63) // 64


def _paths(c, seed):
    """Accepted paths: the first node and up to seven later ones, in order."""
    _, new, _ = _shape(c)
    r = np.random.default_rng(seed + 77)
    got = []
    for n in new:
        k = int(r.integers(1, min(8, n) + 1))
        got.append([0] + sorted(int(x) for x in r.permutation(np.arange(1, n))[: k - 1]))
    return got


# ------------------------------------------------------------------ inputs

_ENGINE = None


def _engine():
    """The program's one engine, set up as a serving loop does."""
    global _ENGINE
    from pagedattentionmetal_amd import PagedAttentionEngine
    if _ENGINE is None:
        _ENGINE = PagedAttentionEngine()
        _ENGINE.set_graceful_degradation(False)
        _ENGINE.set_gpu_timing(False)
        _ENGINE.synchronous = False
    _ENGINE.set_stream(torch.cuda.current_stream())
    return _ENGINE


def _dev(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda", dtype)


def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(mean, std, generator=gen)


def _pool(gen, c, blocks):
    """One pool's contents and, for e4m3, the blocks' scales: N(0, 1) rows with 1% of the entries eight times larger."""
    shape = (blocks, c["block"], c["kv_heads"], c["dim"])
    if c["dtype"] != E4M3:
        return _normal(gen, shape, TORCH[c["dtype"]], 0.5), None
    x = _normal(gen, shape, torch.float16)
    x = x * (1 + 7 * (torch.rand(x.shape, device="cuda", generator=gen) < 0.01)).to(x.dtype)
    s = (x.abs().amax((1, 2, 3)).float() / 448).half()
    q = (x.float() / s.float()[:, None, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(torch.uint8), s


def _batch(c, seed):
    """A batch's lengths, rows, trees and shuffled blocks."""
    ctx, new, parents = _shape(c)
    rng = np.random.default_rng(seed)
    blocks = (ctx + new + c["block"] - 1) // c["block"]
    total = int(blocks.sum())
    flat = rng.permutation(total + 8)[:total]
    width = int(blocks.max())
    bt = np.zeros((len(ctx), width), np.int64)
    bt[np.arange(width)[None, :] < blocks[:, None]] = flat
    rows = int(new.sum())
    at = np.repeat(np.arange(len(new)), new), np.concatenate([np.arange(n) for n in new])
    return dict(ctx=_dev(ctx), new=_dev(new), cu=_dev(np.concatenate([[0], np.cumsum(new)])), bt=_dev(bt),
                flat=_dev(flat), width=width, blocks=total + 8, rows=rows, row_seq=_dev(at[0], torch.int64),
                row_node=_dev(at[1], torch.int64), parents=_dev(parents[at]), nodes=c["nodes_hi"])


def _on_path(parents, seq, node, batch, nodes):
    """[batch, nodes, nodes] truth values: column j is on row i's path (the node itself and its ancestors)."""
    reach = torch.eye(nodes, device="cuda").repeat(batch, 1, 1)
    has = parents >= 0
    reach[seq, node, torch.where(has, parents.long(), node)] = 1.0
    for _ in range(max(1, (nodes - 1).bit_length())):  # paths of twice the length
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _pack(bits):
    """Truth values [rows, 64 w] as w words, bit b of a word its b-th value."""
    b = bits.view(bits.shape[0], -1, 64).long() << torch.arange(64, device="cuda")
    return b.sum(2)


def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = c["kind"]
    if kind in ("rope", "rope_grad"):
        H, K, d, n, t = c["heads"], c["kv_heads"], c["dim"], c["tokens"], TORCH[c["dtype"]]
        s = {"qkv": _normal(gen, (n, (H + 2 * K) * d), t)}  # the projection's packed rows
        s["q"] = s["qkv"][:, : H * d].view(n, H, d)
        s["k"] = s["qkv"][:, H * d: (H + K) * d].view(n, K, d)
        s["v"] = s["qkv"][:, (H + K) * d:].view(n, K, d)
        s["qw"], s["kw"] = (_normal(gen, (d,), t, 0.1, 1.0) for _ in range(2))
        rng = np.random.default_rng(seed)
        s["pos"] = _dev(rng.integers(c["pos_lo"], c["pos_hi"], n))
        r = c["rotary"]
        s["freq"] = BASE ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        if kind == "rope_grad":
            s["dq"], s["dk"] = _normal(gen, (n, H, d), t), _normal(gen, (n, K, d), t)
        elif c["append"]:
            blocks = (n + c["block"] - 1) // c["block"] + 8
            s["slots"] = _dev(rng.permutation(blocks * c["block"])[:n], torch.int64)
            s["kp"], s["vp"] = (torch.zeros((blocks, c["block"], K, d), dtype=t, device="cuda") for _ in range(2))
        return s
    s = _batch(c, seed)
    if kind == "plan":
        return s
    for n in ("k", "v"):
        s[n], s[n + "s"] = _pool(gen, c, s["blocks"])
    if kind == "commit":
        p = _paths(c, seed)
        s["paths"] = _dev(np.array([x + [-1] * (8 - len(x)) for x in p]))
        return s
    s["q"] = _normal(gen, (s["rows"], c["heads"], c["dim"]), torch.float32 if c["dtype"] == F32 else torch.float16)
    on = _on_path(s["parents"], s["row_seq"], s["row_node"], c["batch"], s["nodes"])[s["row_seq"], s["row_node"]]
    s["mask"] = _pack(torch.nn.functional.pad(on, (0, 64 * _words(c) - s["nodes"])))
    return s


def prepare(c, seed):
    s = _inputs(c, seed)
    s["case"] = c
    if own:
        from pagedattentionmetal_amd import PagedLayerSpec, RotarySpec
        s["engine"] = _engine()
        kind = c["kind"]
        if kind == "plan":
            cap = (s["rows"] + 63) // 64 * 64
            new = lambda shape, t=torch.int32: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
            s["out"] = dict(cu_queries=new(c["batch"] + 1), seq_lengths=new(c["batch"]),
                            block_tables=new((c["batch"], s["width"])), positions=new(cap),
                            slot_mapping=new(cap, torch.int64),
                            tree_mask=new((cap, _words(c)), torch.int64) if c["tree"] else None)
        else:
            s["layer"] = PagedLayerSpec(c["dim"], c.get("heads", c["kv_heads"]), c["kv_heads"], c["block"] if
                                        "block" in c else 16, c["dtype"], c.get("window", 0))
        if kind in ("rope", "rope_grad"):
            s["rotary"] = RotarySpec(c["rotary"], BASE, c["interleaved"])
    return s


# ------------------------------------------------------------------ one pass: the framework's calls


def _run_own(s):
    c, e = s["case"], s["engine"]
    kind = c["kind"]
    if kind == "plan":
        e.batch_plan(s["ctx"], s["new"], s["flat"], c["block"], **s["out"], parents=s["parents"] if c["tree"] else None)
        return s["out"]
    if kind == "rope":
        q = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
        if c["append"]:
            e.qk_norm_rope(s["q"], s["k"], q, None, s["pos"], s["layer"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                           rotary=s["rotary"], values=s["v"], k_pool=s["kp"], v_pool=s["vp"], slot_mapping=s["slots"])
            return [q, s["kp"], s["vp"]]
        k = torch.empty_like(s["k"], memory_format=torch.contiguous_format)
        e.qk_norm_rope(s["q"], s["k"], q, k, s["pos"], s["layer"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                       rotary=s["rotary"])
        return [q, k]
    if kind == "rope_grad":
        q = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
        k = torch.empty_like(s["k"], memory_format=torch.contiguous_format)
        qw, kw = (torch.empty(c["dim"], dtype=torch.float32, device="cuda") for _ in range(2))
        e.qk_norm_rope_backward(s["q"], s["k"], s["dq"], s["dk"], q, k, s["pos"], s["layer"], q_weight=s["qw"],
                                k_weight=s["kw"], d_q_weight=qw, d_k_weight=kw, eps=EPS, rotary=s["rotary"])
        return [q, k, qw, kw]
    if kind == "tree":
        out = torch.empty_like(s["q"])
        e.tree_attention(s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["cu"], s["mask"], out, c["nodes_hi"], s["layer"],
                         k_scale=s["ks"], v_scale=s["vs"])
        return out
    lens = torch.empty_like(s["ctx"])
    e.tree_commit(s["k"], s["v"], s["bt"], s["ctx"], s["new"], s["paths"], s["layer"], new_lengths=lens)
    return [lens, s["k"], s["v"]]


# ------------------------------------------------------------------ one pass: the plain form


def _slot_of(bt, seq, pos, block):
    """Pool slots of positions of sequences."""
    return bt.long()[seq, pos // block] * block + pos % block


def _plan(s, c):
    ctx, new, bs = s["ctx"].long(), s["new"].long(), c["block"]
    cap = (s["rows"] + 63) // 64 * 64
    total = ctx + new
    blocks = (total + bs - 1) // bs
    first = torch.cumsum(blocks, 0) - blocks
    col = torch.arange(s["width"], device="cuda")
    at = (first[:, None] + col).clamp(max=s["flat"].numel() - 1)
    bt = torch.where(col < blocks[:, None], s["flat"][at], 0)
    end = torch.cumsum(new, 0)
    cu = torch.cat([torch.zeros_like(end[:1]), end])
    row = torch.arange(cap, device="cuda")
    live = row < end[-1]
    seq = torch.searchsorted(end, row, right=True).clamp(max=len(ctx) - 1)
    node = row - cu[seq]
    out = dict(cu_queries=cu.int(), seq_lengths=total.int(), block_tables=bt.int())
    pos = ctx[seq] + node
    slot = _slot_of(bt, seq, torch.where(live, pos, 0), bs)
    out["slot_mapping"] = torch.where(live, slot, -1)
    out["tree_mask"] = None
    if c["tree"]:
        r = s["rows"]
        on = _on_path(s["parents"], seq[:r], node[:r], len(ctx), s["nodes"])[seq[:r], node[:r]]
        pos = torch.nn.functional.pad(ctx[seq[:r]] + on.sum(1) - 1, (0, cap - r))
        words = _pack(torch.nn.functional.pad(on, (0, 64 * _words(c) - s["nodes"])))
        out["tree_mask"] = torch.nn.functional.pad(words, (0, 0, 0, cap - r))
    out["positions"] = torch.where(live, pos, 0).int()
    return out


def _pairs(x, interleaved):
    """The two halves of every rotated pair."""
    if interleaved:
        return x[..., 0::2], x[..., 1::2]
    return x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]


def _join(a, b, rest, interleaved):
    x = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((x, rest), -1)


def _angles(s):
    a = s["pos"].double()[:, None] * s["freq"]  # far positions: the angle in 64 bits
    return torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]


def _norm_rope(x, w, cos, sin, c):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = _pairs(y[..., : c["rotary"]], c["interleaved"])
    return _join(a * cos - b * sin, b * cos + a * sin, y[..., c["rotary"]:], c["interleaved"])


def _norm_rope_grad(x, w, g, cos, sin, c):
    x, g, w = x.float(), g.float(), w.float()
    a, b = _pairs(g[..., : c["rotary"]], c["interleaved"])
    g = _join(a * cos + b * sin, b * cos - a * sin, g[..., c["rotary"]:], c["interleaved"])
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    h = g * w
    return r * (h - n * (h * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))


def _values(x, scale, dtype):
    """A pool's elements: e4m3 codes stand for code * scale rounded to binary16."""
    if dtype != E4M3:
        return x.float()
    return (x.view(torch.float8_e4m3fn).half() * scale[:, None, None, None]).float()


def _tree(s, c):
    H, K, d, bs, W, n = c["heads"], c["kv_heads"], c["dim"], c["block"], c["window"], s["nodes"]
    B, G, ctx, new = c["batch"], c["heads"] // c["kv_heads"], s["ctx"].long(), s["new"].long()
    L = s["width"] * bs
    k, v = (_values(s[x][s["bt"].long().flatten()], None if s[x + "s"] is None else
                    s[x + "s"][s["bt"].long().flatten()], c["dtype"]).view(B, L, K, d) for x in ("k", "v"))
    q = torch.zeros((B, n, H, d), device="cuda")
    q[s["row_seq"], s["row_node"]] = s["q"].float()
    q = q.view(B, n, K, G, d).permute(0, 2, 1, 3, 4).reshape(B, K, n * G, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(B, K, n, G, L) * (1 / math.sqrt(d))
    # keys a node sees: the cached context and its own path, the last W of them
    words = torch.zeros((B, n, _words(c)), dtype=torch.int64, device="cuda")
    words[s["row_seq"], s["row_node"]] = s["mask"]
    on = ((words[..., None] >> torch.arange(64, device="cuda")) & 1).flatten(2)[..., :n].bool()
    j = torch.arange(L, device="cuda")
    past = (j < ctx[:, None])[:, None].expand(B, n, L)
    drafted = (j >= ctx[:, None]) & (j < (ctx + new)[:, None])
    node = (j - ctx[:, None]).clamp(0, n - 1)
    see = past | (drafted[:, None] & torch.gather(on, 2, node[:, None].expand(B, n, L)))
    if W:
        rank = torch.cumsum(see, 2)
        see = see & (rank > rank[..., -1:] - W)
    see = see[:, None, :, None]
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)  # a row that sees no key is zeros
    seen = see.any(2).any(2)[:, 0, :, None, None]  # keys that no row sees are not read
    o = torch.matmul(p.view(B, K, n * G, L), torch.where(seen, v, 0.0).permute(0, 2, 1, 3).contiguous())
    o = o.view(B, K, n, G, d).permute(0, 2, 1, 3, 4).reshape(B, n, H, d)
    return o[s["row_seq"], s["row_node"]].to(s["q"].dtype)


def _commit(s, c):
    ctx, path = s["ctx"].long(), s["paths"].long()
    k = torch.arange(path.shape[1], device="cuda")
    k = torch.minimum(k, s["new"].long()[:, None] - 1)
    live = path >= 0
    seq = torch.arange(len(ctx), device="cuda")[:, None].expand(path.shape)
    dst = _slot_of(s["bt"], seq, ctx[:, None] + k, c["block"])
    src = torch.where(live, _slot_of(s["bt"], seq, ctx[:, None] + path.clamp(min=0), c["block"]), dst)
    for x in ("k", "v"):
        flat = s[x].view(-1, c["kv_heads"] * c["dim"])
        flat[dst] = flat[src]
    return [(ctx + live.sum(1)).int(), s["k"], s["v"]]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    kind = c["kind"]
    if kind == "plan":
        return _plan(s, c)
    if kind == "tree":
        return _tree(s, c)
    if kind == "commit":
        return _commit(s, c)
    t = TORCH[c["dtype"]]
    cos, sin = _angles(s)
    if kind == "rope_grad":
        dq, dqw = _norm_rope_grad(s["q"], s["qw"], s["dq"], cos, sin, c)
        dk, dkw = _norm_rope_grad(s["k"], s["kw"], s["dk"], cos, sin, c)
        return [dq.to(t), dk.to(t), dqw, dkw]
    q, k = (_norm_rope(s[x], s[x + "w"], cos, sin, c).to(t) for x in ("q", "k"))
    if not c["append"]:
        return [q, k]
    s["kp"].view(-1, c["kv_heads"], c["dim"])[s["slots"]] = k
    s["vp"].view(-1, c["kv_heads"], c["dim"])[s["slots"]] = s["v"]
    return [q, s["kp"], s["vp"]]


# ------------------------------------------------------------------ 64 bits


def _rope64(x, w, pos, c):
    x = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w
    r = c["rotary"]
    f = torch.exp(torch.arange(r // 2, device="cuda", dtype=torch.float64) * (-2.0 / r * math.log(BASE)))
    turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64), torch.outer(pos.double(), f))[:, None]
    head = x[..., :r]
    z = head.unflatten(-1, (r // 2, 2)) if c["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, x[..., r:]], -1)


def _tree64(s, c):
    H, K, d, bs = c["heads"], c["kv_heads"], c["dim"], c["block"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (C, n) in enumerate(zip(s["ctx"].tolist(), s["new"].tolist())):
        j = torch.arange(C + n, device="cuda")
        phys = s["bt"][b].long()[j // bs]
        kv = []
        for x in ("k", "v"):
            y = s[x][phys, j % bs]
            if c["dtype"] == E4M3:
                y = y.view(torch.float8_e4m3fn).half() * s[x + "s"][phys][:, None, None]
            kv.append(y.double())
        see = np.ones((n, C + n), bool)
        for i in range(n):
            w = [int(x) & (1 << 64) - 1 for x in s["mask"][row + i].tolist()]
            see[i, C:] = [w[m // 64] >> m % 64 & 1 for m in range(n)]
            if c["window"]:
                keys = np.flatnonzero(see[i])
                see[i, keys[:max(0, len(keys) - c["window"])]] = False
        hide = ~torch.from_numpy(see).to("cuda")
        empty = hide.all(1)
        for h in range(H):
            g = h * K // H
            q = s["q"][row: row + n, h].double()
            x = (q @ kv[0][:, g].t().contiguous()) / math.sqrt(d)
            x = torch.softmax(x.masked_fill(hide, -math.inf), 1).masked_fill(empty[:, None], 0.0)
            out[row: row + n, h] = x @ kv[1][:, g].contiguous()
        row += n
    return out


def exact(c, seed):
    kind = c["kind"]
    if kind == "plan":  # whole numbers
        return None
    s = _inputs(c, seed)
    if kind == "tree":
        return _tree64(s, c)
    if kind == "commit":
        out = [None]
        for x in ("k", "v"):
            p = s[x].double().cpu()
            for b, path in enumerate(_paths(c, seed)):
                bt, C = s["bt"][b].tolist(), int(s["ctx"][b])
                for i, m in enumerate(path):
                    to, of = C + i, C + m
                    p[bt[to // c["block"]], to % c["block"]] = p[bt[of // c["block"]], of % c["block"]].clone()
            out.append(p)
        return out
    x = {n: s[n].double().clone().requires_grad_() for n in ("q", "k", "qw", "kw")}
    q, k = _rope64(x["q"], x["qw"], s["pos"], c), _rope64(x["k"], x["kw"], s["pos"], c)
    if kind == "rope_grad":
        return list(torch.autograd.grad([q, k], [x["q"], x["k"], x["qw"], x["kw"]], [s["dq"].double(), s["dk"].double()]))
    if not c["append"]:
        return [q.detach(), k.detach()]
    out = [q.detach()]
    for p, rows in ((s["kp"], k.detach()), (s["vp"], s["v"].double())):
        y = torch.zeros(p.shape, dtype=torch.float64, device="cuda").view(-1, c["kv_heads"], c["dim"])
        y[s["slots"]] = rows
        out.append(y.view(p.shape))
    return out
