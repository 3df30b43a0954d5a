"""The speculative-decoding calls on the GPU: batch plans, norm and rotation of query and key heads with their
gradients, tree attention and commits, against plain implementations in 64 bits, and a step of all of them together,
eager and captured.

Tolerances count roundings.  u = 2^-24 is half a step of binary32, h = 2^-11 of binary16.
"""
import numpy as np
import pytest

from helpers import to_dev, to_host

pytestmark = pytest.mark.gpu

U, HALF = 2.0 ** -24, 2.0 ** -11
NP = {0: np.float32, 1: np.float16, 2: np.float16}


def _engine():
    from pagedattentionmetal_amd import PagedAttentionEngine
    e = PagedAttentionEngine()
    e.set_graceful_degradation(False)
    return e


def _layer(d, H, K, bs=16, dtype=1, window=0):
    from pagedattentionmetal_amd import PagedLayerSpec
    return PagedLayerSpec(d, H, K, bs, dtype, window)


def _i32(x):
    return to_dev(np.asarray(x, np.int32))


def _tree(rng, n, chain=0.5):
    """Parents of a random tree of n nodes: -1 for roots, a few of them."""
    return np.array([-1 if i == 0 or rng.random() < 0.05 else (i - 1 if rng.random() < chain else rng.integers(0, i))
                     for i in range(n)], np.int32)


def _paths(parents):
    on = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            on[i] = on[p]
        on[i, i] = True
    return on


def _words(on, words):
    out = np.zeros((on.shape[0], words), np.uint64)
    for i, j in zip(*np.nonzero(on)):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


# ------------------------------------------------------------------ batch plan


def _plan_ref(ctx, new, flat, bs, width, cap, parents, words):
    n = len(ctx)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    bt = np.zeros((n, width), np.int32)
    pos, slot = np.zeros(cap, np.int32), np.full(cap, -1, np.int64)
    mask = np.zeros((cap, max(1, words)), np.uint64)
    first = 0
    for s in range(n):
        L = ctx[s] + new[s]
        nb = -(-L // bs)
        bt[s, :nb] = flat[first:first + nb]
        on = _paths(parents[cu[s]:cu[s + 1]]) if parents is not None else np.tril(np.ones((new[s], new[s]), bool))
        for i in range(new[s]):
            t = ctx[s] + i
            slot[cu[s] + i] = int(flat[first + t // bs]) * bs + t % bs
            pos[cu[s] + i] = ctx[s] + on[i].sum() - 1
        if words:
            mask[cu[s]:cu[s + 1]] = _words(on, words)
        first += nb
    return cu.astype(np.int32), (np.asarray(ctx) + new).astype(np.int32), bt, pos, slot, mask


def _plan(eng, ctx, new, flat, bs, width, cap, parents=None, words=0, status=False):
    import torch
    n = len(ctx)
    fill = lambda shape, t=torch.int32: torch.full(shape, 77, dtype=t, device="cuda")  # noqa: E731
    out = dict(cu_queries=fill((n + 1,)), seq_lengths=fill((n,)), block_tables=fill((n, width)), positions=fill((cap,)),
               slot_mapping=fill((cap,), torch.int64), tree_mask=fill((cap, words), torch.int64) if words else None,
               status=torch.zeros(1, dtype=torch.int32, device="cuda") if status else None)
    eng.batch_plan(_i32(ctx), _i32(new), _i32(flat), bs, parents=None if parents is None else _i32(parents), **out)
    return {k: None if v is None else to_host(v) for k, v in out.items()}


@pytest.mark.parametrize("n,bs,ctx_hi,new_hi,tree,words,extra", [
    (1, 16, 0, 1, False, 0, 0),          # one token of an empty sequence
    (3, 16, 100, 8, True, 1, 5),
    (5, 1, 40, 64, True, 1, 64),         # one-token blocks, full mask words
    (7, 12, 300, 130, True, 3, 1),       # words that are not full, a block size between powers of two
    (4, 16, 20000, 700, False, 11, 0),   # several workgroups a sequence
    (300, 8, 64, 3, False, 1, 9),
    (2500, 16, 40, 2, True, 1, 30),      # several sequences a workgroup
    (2, 16, 5, 1024, True, 16, 0),       # the largest tree
    (6, 16, 50, 0, False, 0, 4),         # no new tokens at all
])
def test_batch_plan(n, bs, ctx_hi, new_hi, tree, words, extra):
    rng = np.random.default_rng(n * 31 + bs)
    ctx, new = rng.integers(0, ctx_hi + 1, n), rng.integers(0, new_hi + 1, n)
    if new_hi == 1024:
        new[0] = 1024
    if n == 1:
        new[0] = 1
    parents = np.concatenate([_tree(rng, k) for k in new] + [np.zeros(0, np.int32)]) if tree else None
    blocks = -(-(ctx + new) // bs)
    flat = rng.permutation(int(blocks.sum()) + 5)
    width, cap = max(1, int(blocks.max())) + 2, max(1, int(new.sum())) + extra
    got = _plan(_engine(), ctx, new, flat, bs, width, cap, parents, words, status=True)
    cu, lens, bt, pos, slot, mask = _plan_ref(ctx, new, flat, bs, width, cap, parents, words)
    assert got["status"][0] == 0
    for name, ref in (("cu_queries", cu), ("seq_lengths", lens), ("block_tables", bt), ("positions", pos),
                      ("slot_mapping", slot)):
        assert np.array_equal(got[name], ref), name
    if words:
        assert np.array_equal(got["tree_mask"].view(np.uint64), mask)


def test_batch_plan_that_does_not_fit_stays_inside_its_buffers():
    """Rows past max_rows, blocks past the table and past the list, negative lengths, bad parents: reported by their
    bits, nothing written outside."""
    import torch
    eng = _engine()
    bs = 4
    # two sequences of 6 + 3 tokens (3 blocks each)
    g = _plan(eng, [6, 6], [3, 3], np.arange(10, 16), bs, 3, 5, status=True)
    assert g["status"][0] == 1 and g["cu_queries"].tolist() == [0, 3, 5]
    assert g["slot_mapping"].tolist() == [46, 47, 48, 58, 59]
    g = _plan(eng, [6, 6], [3, 3], np.arange(10, 16), bs, 2, 6, status=True)
    assert g["status"][0] == 2 and g["block_tables"].tolist() == [[10, 11], [13, 14]]
    assert g["slot_mapping"].tolist() == [46, 47, -1, 58, 59, -1] and g["seq_lengths"].tolist() == [8, 8]
    g = _plan(eng, [6, 6], [3, 3], np.arange(10, 15), bs, 3, 6, status=True)
    assert g["status"][0] == 2 and g["block_tables"].tolist() == [[10, 11, 12], [13, 14, 0]]
    assert g["slot_mapping"].tolist() == [46, 47, 48, 58, 59, -1]
    g = _plan(eng, [-6, 2], [1, -3], np.arange(10, 16), bs, 3, 6, status=True)
    assert g["status"][0] == 4 and g["cu_queries"].tolist() == [0, 1, 1] and g["seq_lengths"].tolist() == [1, 2]
    # parents that name themselves, a later node, or nothing; a list that is too short
    g = _plan(eng, [6], [5], np.arange(10, 16), bs, 3, 5, parents=[-1, 1, 4, -7], words=1, status=True)
    assert g["status"][0] == 8 and g["tree_mask"][:, 0].tolist() == [1, 2, 4, 8, 16]
    assert g["positions"].tolist() == [6] * 5
    # a tree past its mask's words
    g = _plan(eng, [0], [70], np.arange(10, 30), bs, 18, 70, parents=np.arange(-1, 69), words=1, status=True)
    assert g["status"][0] == 8 and (g["slot_mapping"][64:] == -1).all() and (g["slot_mapping"][:64] >= 0).all()
    assert (g["tree_mask"][64:] == 0).all()
    big = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert int(big) == 0  # the device is well


# ------------------------------------------------------------------ norm and rotation


def _rope64(x, w, pos, rotary, interleaved, inv_freq, eps, normalize):
    """[n, h, d] in 64 bits; also the norm's output before the rotation."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if normalize else x.copy()
    if w is not None:
        y = y * w.astype(np.float64)
    out = y.copy()
    if rotary:
        a = pos.astype(np.float64)[:, None] * np.asarray(inv_freq)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        i = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2),
                                                                           slice(rotary // 2, rotary))
        out[..., i[0]] = y[..., i[0]] * c - y[..., i[1]] * s
        out[..., i[1]] = y[..., i[1]] * c + y[..., i[0]] * s
    return out, y


def _step(dtype, ref):
    """Half a step of the type at the values: binary16 also below its normal range."""
    return np.abs(ref) * U if dtype == 0 else np.maximum(np.abs(ref) * HALF, 2.0 ** -25)


def _rope_tol(dtype, y, ref):
    """A row's sum of squares adds at most 16 products a lane and 6 levels of lanes (22 roundings, half of them after
    the root), the root, quotient and two products 5, cosine and sine 2 (their Taylor sums are within 2e-9) and the
    rotation 2: at most 32 u of the larger of a pair, twice for its two products."""
    return 64 * U * np.abs(y).max(-1, keepdims=True) + _step(dtype, ref)


NORM_CASES = [
    # dtype, n, H, K, d, rotary, interleaved, normalize, weights
    (1, 5, 8, 2, 128, 128, False, True, True),
    (1, 64, 32, 8, 128, 128, False, True, True),
    (0, 33, 4, 4, 128, 64, True, True, True),
    (1, 3, 6, 2, 96, 96, False, True, True),     # 6 lanes of 8
    (0, 7, 3, 1, 80, 80, True, True, True),
    (1, 17, 12, 4, 80, 40, False, True, False),  # halves of 20: single pairs
    (0, 9, 5, 5, 36, 22, False, True, True),     # an odd count of pairs
    (1, 1, 1, 1, 4, 4, True, True, True),
    (0, 2, 2, 2, 256, 256, False, True, True),
    (1, 4, 2, 1, 252, 126, True, True, True),    # more units than lanes
    (1, 11, 8, 2, 64, 0, False, True, True),     # norm alone
    (0, 13, 8, 2, 64, 64, False, False, False),  # rotation alone
    (1, 1000, 2, 1, 256, 128, True, True, True),
    (1, 4000, 4, 1, 64, 64, False, True, True),  # several tokens a workgroup
]


@pytest.mark.parametrize("dtype,n,H,K,d,rotary,inter,normalize,weights", NORM_CASES)
def test_qk_norm_rope(dtype, n, H, K, d, rotary, inter, normalize, weights):
    import torch
    from pagedattentionmetal_amd import RotarySpec
    rng = np.random.default_rng(n + d)
    dt = NP[dtype]
    qkv = rng.standard_normal((n, (H + 2 * K) * d)).astype(dt)  # packed projections, read in place
    qkv[0] *= 0 if n > 2 else 1  # a row of zeros
    pos = rng.integers(0, 5000, n).astype(np.int32)
    pos[-1] = 2 ** 31 - 1 if n > 2 else 7
    qw, kw = (rng.normal(1, 0.2, d).astype(dt) for _ in range(2)) if weights else (None, None)
    rot = RotarySpec(rotary, 10000.0, inter)
    dev = to_dev(qkv)
    q, k = dev[:, : H * d].view(n, H, d), dev[:, H * d:(H + K) * d].view(n, K, d)
    qo = torch.full((n, H, d), 9.0, dtype=q.dtype, device="cuda")
    ko = torch.full((n, K, d), 9.0, dtype=q.dtype, device="cuda")
    _engine().qk_norm_rope(q, k, qo, ko, _i32(pos), _layer(d, H, K, 16, dtype), q_weight=None if qw is None else
                           to_dev(qw), k_weight=None if kw is None else to_dev(kw), eps=1e-5, rotary=rot,
                           normalize=normalize)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        ref, y = _rope64(to_host(x), w, pos, rotary, inter, rot.inv_freq, 1e-5, normalize)
        err = np.abs(to_host(got).astype(np.float64) - ref)
        assert (err <= _rope_tol(dtype, y, ref)).all(), float((err - _rope_tol(dtype, y, ref)).max())


@pytest.mark.parametrize("dtype,shift", [(1, 0), (1, 1), (0, 1)])
def test_qk_norm_rope_in_place_and_unaligned(dtype, shift):
    """In place, at an address that is no whole piece (shift elements off)."""
    from pagedattentionmetal_amd import RotarySpec
    rng = np.random.default_rng(5)
    n, H, K, d = 21, 4, 2, 128
    base = to_dev(rng.standard_normal(shift + n * 1000).astype(NP[dtype]))
    rows = base[shift:].view(n, 1000)
    q, k = rows[:, : H * d].view(n, H, d), rows[:, H * d:(H + K) * d].view(n, K, d)
    pos = np.arange(n).astype(np.int32) * 100000
    rot = RotarySpec(128, 500000.0)
    before, rest = (to_host(q).copy(), to_host(k).copy()), to_host(rows[:, (H + K) * d:]).copy()
    _engine().qk_norm_rope(q, k, q, k, _i32(pos), _layer(d, H, K, 16, dtype), rotary=rot)
    for x, b in ((q, before[0]), (k, before[1])):
        ref, y = _rope64(b, None, pos, 128, False, rot.inv_freq, 1e-6, True)
        assert (np.abs(to_host(x).astype(np.float64) - ref) <= _rope_tol(dtype, y, ref)).all()
    assert np.array_equal(to_host(rows[:, (H + K) * d:]), rest)


@pytest.mark.parametrize("dtype,n,d,keep", [(1, 70, 128, True), (0, 9, 64, False), (1, 33, 20, False)])
def test_qk_norm_rope_into_the_pools(dtype, n, d, keep):
    """Keys and values to their slots; negative slots and slots past the pools are not written."""
    import torch
    from pagedattentionmetal_amd import RotarySpec
    rng = np.random.default_rng(n)
    H, K, bs, nb = 8, 2, 16, 12
    dt = NP[dtype]
    q, k, v = (to_dev(rng.standard_normal((n, h, d)).astype(dt)) for h in (H, K, K))
    pos = rng.integers(0, 1000, n).astype(np.int32)
    slots = rng.permutation(nb * bs)[:n].astype(np.int64)
    slots[1], slots[2], slots[-1] = -1, nb * bs, 1 << 40
    kp, vp = (torch.full((nb, bs, K, d), 5.0, dtype=q.dtype, device="cuda") for _ in range(2))
    qo = torch.empty_like(q)
    ko = torch.empty_like(k) if keep else None
    rot = RotarySpec(d, 10000.0)
    _engine().qk_norm_rope(q, k, qo, ko, _i32(pos), _layer(d, H, K, bs, dtype), rotary=rot, values=v, k_pool=kp,
                           v_pool=vp, slot_mapping=to_dev(slots))
    ref, y = _rope64(to_host(k), None, pos, d, False, rot.inv_freq, 1e-6, True)
    ok = (slots >= 0) & (slots < nb * bs)
    rk, rv = to_host(kp).reshape(-1, K, d), to_host(vp).reshape(-1, K, d)
    assert (np.abs(rk[slots[ok]].astype(np.float64) - ref[ok]) <= _rope_tol(dtype, y, ref)[ok]).all()
    assert np.array_equal(rv[slots[ok]], to_host(v)[ok])
    rest = np.setdiff1d(np.arange(nb * bs), slots[ok])
    assert (rk[rest] == 5).all() and (rv[rest] == 5).all()
    if keep:
        assert np.array_equal(to_host(ko)[ok], rk[slots[ok]])
        assert (np.abs(to_host(ko).astype(np.float64) - ref) <= _rope_tol(dtype, y, ref)).all()


def _rope_grad64(x, w, g, pos, rotary, interleaved, inv_freq, eps, normalize):
    x, g = x.astype(np.float64), g.astype(np.float64)
    g, _ = _rope64(g, None, pos, rotary, interleaved, -np.asarray(inv_freq), 0.0, False)
    if not normalize:
        return g, None, g, np.abs(g)
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, h = x * r, g * w
    dx = r * (h - n * (h * n).mean(-1, keepdims=True))
    # what the sums' roundings are measured by
    size = r * (np.abs(h).max(-1, keepdims=True) + np.abs(n).max(-1, keepdims=True) * np.abs(h * n).mean(-1, keepdims=True))
    return dx, (g * n).sum((0, 1)), size, np.abs(g * n).sum((0, 1))


@pytest.mark.parametrize("dtype,n,H,K,d,rotary,inter,normalize,weights", NORM_CASES)
def test_qk_norm_rope_backward(dtype, n, H, K, d, rotary, inter, normalize, weights):
    """dx: the rotation's and norm's roundings (64 u of a row's size, as in the forward, and as many again for the
    row's sum of products) and the output's.  dw: a lane adds the rows it meets one after another (at most n H), a row's
    term carries the forward's 32 roundings, and the groups' sums 20 levels."""
    import torch
    from pagedattentionmetal_amd import RotarySpec
    rng = np.random.default_rng(n + d + 1)
    dt = NP[dtype]
    qkv = rng.standard_normal((n, (H + K) * d)).astype(dt)
    pos = rng.integers(0, 5000, n).astype(np.int32)
    qw, kw = (rng.normal(1, 0.2, d).astype(dt) for _ in range(2)) if weights else (None, None)
    gq, gk = rng.standard_normal((n, H, d)).astype(dt), rng.standard_normal((n, K, d)).astype(dt)
    rot = RotarySpec(rotary, 10000.0, inter)
    dev = to_dev(qkv)
    q, k = dev[:, : H * d].view(n, H, d), dev[:, H * d:].view(n, K, d)
    dq, dk = torch.full((n, H, d), 9.0, dtype=q.dtype, device="cuda"), torch.full((n, K, d), 9.0, dtype=q.dtype,
                                                                                    device="cuda")
    dqw, dkw = (torch.full((d,), 9.0, device="cuda") if normalize else None for _ in range(2))
    eng = _engine()
    args = (q, k, to_dev(gq), to_dev(gk), dq, dk, _i32(pos), _layer(d, H, K, 16, dtype))
    kw_ = dict(q_weight=None if qw is None else to_dev(qw), k_weight=None if kw is None else to_dev(kw), d_q_weight=dqw,
               d_k_weight=dkw, eps=1e-5, rotary=rot, normalize=normalize)
    eng.qk_norm_rope_backward(*args, **kw_)
    for got, gotw, x, w, g, heads in ((dq, dqw, q, qw, gq, H), (dk, dkw, k, kw, gk, K)):
        dx, dw, size, total = _rope_grad64(to_host(x), w, g, pos, rotary, inter, rot.inv_freq, 1e-5, normalize)
        err = np.abs(to_host(got).astype(np.float64) - dx)
        assert (err <= 128 * U * np.abs(size).max(-1, keepdims=True) + _step(dtype, dx)).all()
        if normalize:
            assert (np.abs(to_host(gotw).astype(np.float64) - dw) <= (min(n * heads, 256) + 52) * U * total + 1e-30).all()
    first = [None if t is None else to_host(t).copy() for t in (dq, dk, dqw, dkw)]
    eng.qk_norm_rope_backward(*args, **kw_)
    for a, t in zip(first, (dq, dk, dqw, dkw)):
        assert a is None or np.array_equal(a, to_host(t)), "the same bits every time"


def test_qk_norm_rope_backward_by_differences():
    """The f32 gradient along random directions against central differences of the f64 forward (step 1e-5: the
    difference's own error is about 1e-9 of the loss, the call's 1e-6)."""
    import torch
    from pagedattentionmetal_amd import RotarySpec
    rng = np.random.default_rng(3)
    n, H, K, d = 6, 4, 2, 64
    q, k, gq, gk = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (H, K, H, K))
    qw, kw = (rng.normal(1, 0.2, d).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 3000, n).astype(np.int32)
    rot = RotarySpec(48, 10000.0, True)
    dq, dk = torch.empty(n, H, d, device="cuda"), torch.empty(n, K, d, device="cuda")
    dqw, dkw = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    _engine().qk_norm_rope_backward(to_dev(q), to_dev(k), to_dev(gq), to_dev(gk), dq, dk, _i32(pos),
                                    _layer(d, H, K, 16, 0), q_weight=to_dev(qw), k_weight=to_dev(kw), d_q_weight=dqw,
                                    d_k_weight=dkw, eps=1e-5, rotary=rot)

    def loss(x, w, g):
        return (_rope64(x, w, pos, 48, True, rot.inv_freq, 1e-5, True)[0] * g).sum()
    for x, w, g, dx, dw in ((q, qw, gq, dq, dqw), (k, kw, gk, dk, dkw)):
        for _ in range(3):
            tx, tw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)
            diff = (_f64(loss, x, tx, w, tw, g, 1e-5) - _f64(loss, x, tx, w, tw, g, -1e-5)) / 2e-5
            got = (to_host(dx).astype(np.float64) * tx).sum() + (to_host(dw).astype(np.float64) * tw).sum()
            scale = (np.abs(to_host(dx)) * np.abs(tx)).sum() + (np.abs(to_host(dw)) * np.abs(tw)).sum()
            assert abs(got - diff) <= 2e-6 * scale


def _f64(loss, x, tx, w, tw, g, e):
    x, w = x.astype(np.float64) + e * tx, w.astype(np.float64) + e * tw
    return loss(x, w, g.astype(np.float64))


# ------------------------------------------------------------------ tree attention


class Batch:
    """A ragged batch of drafted trees over shuffled pools, and its attention in 64 bits."""

    def __init__(self, rng, dtype, ctx, new, H, K, d, bs, window=0, words=1, masks="tree", std=1.0, spare=0):
        import torch
        self.dtype, self.ctx, self.new, self.H, self.K, self.d, self.bs, self.window = dtype, ctx, new, H, K, d, bs, window
        n = len(ctx)
        blocks = [-(-(c + t) // bs) for c, t in zip(ctx, new)]
        self.nb, self.width = sum(blocks) + 3, max(1, max(blocks)) + spare
        perm = rng.permutation(self.nb)
        self.bt = np.full((n, self.width), -(1 << 31), np.int32)  # entries past the blocks are never used
        at = 0
        for s, b in enumerate(blocks):
            self.bt[s, :b] = perm[at:at + b]
            at += b
        self.rows = int(sum(new))
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        shape = (self.nb, bs, K, d)
        self.k, self.v = (rng.standard_normal(shape).astype(NP[dtype]) * NP[dtype](std) for _ in range(2))
        self.ks = self.vs = None
        if dtype == 2:
            self.codes, self.scales = [], []
            for x in (self.k, self.v):
                s = (np.abs(x.astype(np.float32)).max((1, 2, 3)) / 448).astype(np.float16)
                c = torch.from_numpy(x.astype(np.float32) / s.astype(np.float32)[:, None, None, None])
                c = c.clamp(-448, 448).to(torch.float8_e4m3fn)
                self.codes.append(c.view(torch.uint8).numpy())
                self.scales.append(s)
            self.k, self.v = ((torch.from_numpy(c).view(torch.float8_e4m3fn).half().numpy() * s[:, None, None, None])
                              for c, s in zip(self.codes, self.scales))
        self.q = rng.standard_normal((self.rows, H, d)).astype(NP[dtype])
        self.see, self.words = [], words
        for s in range(n):
            t = new[s]
            if masks == "chain":
                on = np.tril(np.ones((t, t), bool))
            elif masks == "tree":
                on = _paths(_tree(rng, t))
            else:  # any bits, some rows without
                on = rng.random((t, t)) < 0.4
                on[rng.random(t) < 0.3] = False
            self.see.append(on)
        self.mask = None
        if masks != "chain":
            self.mask = np.zeros((max(1, self.rows), words), np.uint64)
            for s in range(n):
                m = _words(self.see[s], words)
                if new[s] < 64 * words:  # bits past the sequence's nodes say nothing
                    m[:, new[s] // 64] |= np.uint64((0xFFFFFFFFFFFFFFFF << (new[s] % 64)) & 0xFFFFFFFFFFFFFFFF)
                self.mask[self.cu[s]:self.cu[s + 1]] = m

    def slot(self, s, j):
        return self.bt[s, j // self.bs], j % self.bs

    def run(self, eng, out=None, max_queries=None, k=None, v=None, q=None):
        import torch
        kd = to_dev((self.k if k is None else k) if self.dtype != 2 else self.codes[0])
        vd = to_dev((self.v if v is None else v) if self.dtype != 2 else self.codes[1])
        ks, vs = (to_dev(x.view(np.uint16)) for x in self.scales) if self.dtype == 2 else (None, None)
        qd = to_dev(self.q if q is None else q)
        if out is None:
            out = torch.full(qd.shape, 7.0, dtype=qd.dtype, device="cuda")
        eng.tree_attention(qd, kd, vd, _i32(self.bt), _i32(self.ctx), _i32(self.cu), None if self.mask is None else
                           to_dev(self.mask.view(np.int64)), out, max_queries or max(1, max(self.new)),
                           _layer(self.d, self.H, self.K, self.bs, self.dtype, self.window), k_scale=ks, v_scale=vs)
        return to_host(out)

    def visible(self, s):
        """[rows, keys] truth values."""
        c, t = self.ctx[s], self.new[s]
        see = np.ones((t, c + t), bool)
        see[:, c:] = self.see[s]
        if self.window:
            for i in range(t):
                keys = np.flatnonzero(see[i])
                see[i, keys[: max(0, len(keys) - self.window)]] = False
        return see

    def exact(self, q=None, k=None, v=None):
        """Outputs [rows, H, d], and for every row the largest |v| it sees and its scores' error bound."""
        q = (self.q if q is None else q).astype(np.float64)
        out, vmax, ds = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
        k, v = (self.k if k is None else k).astype(np.float64), (self.v if v is None else v).astype(np.float64)
        G = self.H // self.K
        for s in range(len(self.ctx)):
            L = self.ctx[s] + self.new[s]
            j = np.arange(L)
            kk, vv = k[self.bt[s, j // self.bs], j % self.bs], v[self.bt[s, j // self.bs], j % self.bs]
            see = self.visible(s)
            for i in range(self.new[s]):
                r = self.cu[s] + i
                on = see[i]
                if not on.any():
                    continue
                for h in range(self.H):
                    kh, vh = kk[on, h // G], vv[on, h // G]
                    x = kh @ q[r, h] / np.sqrt(self.d)
                    with np.errstate(invalid="ignore"):
                        p = np.exp(x - x.max())
                        out[r, h] = (p[:, None] * vh).sum(0) / p.sum()
                        vmax[r, h] = np.abs(vh).max()
                        ds[r, h] = (np.abs(kh) @ np.abs(q[r, h])).max() / np.sqrt(self.d)
        return out, vmax, ds

    def tolerance(self, ref, vmax, ds):
        """A score's d products add in at most d / 4 + 8 roundings of the sum of magnitudes ds, and scaling and the
        exponential's argument 4 more; a probability is off by that (as e^x) and, relatively, by 8 u; f16 and e4m3
        calls may round it to binary16.  Numerator and denominator: twice, of the largest |v|; sums of p over L keys
        in f32 add 64 u; then the output's rounding."""
        p = 2 * ((self.d / 4 + 12) * U * ds + 8 * U) + 64 * U + (0 if self.dtype == 0 else 2 * HALF)
        return (p * vmax)[..., None] + _step(self.dtype, ref)

    def check(self, got, **kw):
        ref, vmax, ds = self.exact(**kw)
        err, tol = np.abs(got.astype(np.float64) - ref), self.tolerance(ref, vmax, ds)
        bad = ~(err <= tol)
        assert not bad.any(), (np.argwhere(bad)[:5].tolist(), float(err[bad].max()) if bad.any() else 0, int(bad.sum()))


TREE_CASES = [
    # dtype, ctx, new, H, K, d, bs, window, words, masks
    (1, [0], [1], 8, 2, 128, 16, 0, 1, "tree"),                       # one key
    (1, [0], [1], 8, 2, 128, 16, 0, 1, "any"),                        # perhaps none
    (1, [100, 0, 17], [8, 5, 1], 32, 8, 128, 16, 0, 1, "tree"),
    (1, [63, 64, 65], [64, 63, 2], 8, 2, 64, 16, 0, 1, "tree"),       # tiles that end at, before and past the drafts
    (1, [1000, 300], [33, 7], 16, 4, 128, 8, 0, 1, "any"),
    (1, [700, 5], [100, 129], 8, 2, 128, 16, 0, 3, "tree"),           # masks of several words
    (1, [300, 40], [40, 20], 4, 4, 64, 32, 50, 1, "any"),             # windows inside the context
    (1, [20, 3], [40, 64], 8, 1, 128, 16, 9, 1, "tree"),              # windows shorter than the paths
    (1, [50], [30], 8, 2, 128, 16, 1, 1, "tree"),                     # a window of one key
    (1, [90, 10, 0, 33], [3, 0, 2, 1], 12, 4, 96, 16, 0, 1, "tree"),  # a sequence without rows
    (1, [200], [50], 34, 2, 80, 12, 0, 1, "tree"),                    # 17 heads a kv head, odd blocks
    (1, [77], [9], 4, 2, 20, 16, 0, 1, "any"),                        # head sizes that are no whole pieces
    (1, [500], [31], 16, 16, 256, 16, 0, 1, "tree"),
    (1, [2000, 1, 600], [16, 60, 33], 64, 8, 128, 16, 0, 1, "tree"),
    (1, [400, 9], [20, 70], 8, 2, 128, 64, 0, 2, "chain"),
    (0, [100, 0, 17], [8, 5, 1], 8, 2, 128, 16, 0, 1, "tree"),
    (0, [63, 500], [64, 30], 8, 8, 64, 8, 0, 1, "any"),
    (0, [300, 7], [70, 9], 6, 2, 36, 16, 25, 2, "tree"),
    (0, [300, 7], [20, 9], 4, 1, 256, 1, 0, 1, "tree"),
    (0, [1500], [12], 8, 2, 96, 16, 0, 1, "chain"),
    (2, [100, 0, 17], [8, 5, 1], 32, 8, 128, 16, 0, 1, "tree"),
    (2, [63, 900], [64, 30], 8, 2, 64, 16, 0, 1, "any"),
    (2, [300, 7], [70, 9], 6, 2, 96, 16, 25, 2, "tree"),
    (2, [44], [9], 4, 2, 12, 4, 0, 1, "tree"),
    (2, [1500, 20], [32, 32], 64, 8, 128, 16, 600, 1, "tree"),
]


@pytest.mark.parametrize("dtype,ctx,new,H,K,d,bs,window,words,masks", TREE_CASES)
def test_tree_attention(dtype, ctx, new, H, K, d, bs, window, words, masks):
    b = Batch(np.random.default_rng(sum(ctx) + d + H), dtype, ctx, new, H, K, d, bs, window, words, masks, spare=2)
    eng = _engine()
    b.check(b.run(eng))
    assert eng.last_stats["operation"] == 11


MORE_TREE_CASES = [
    (2, [4000, 100], [64, 50], 8, 2, 128, 16, 0, 1, "tree"),                     # e4m3, blocks of 256 rows
    (2, [900], [64], 8, 2, 64, 16, 0, 1, "any"),
    (2, [250, 9], [64, 63], 8, 1, 96, 32, 70, 1, "tree"),
    (2, [500, 30, 2], [64, 20, 7], 8, 2, 128, 16, 0, 1, "tree"),                 # of 128
    (2, [333], [50], 8, 4, 64, 16, 0, 1, "any"),                                 # of 64, two of them
    (2, [300], [40], 8, 2, 72, 16, 0, 1, "tree"),                                # heads of half pieces
    (2, [300], [40], 8, 2, 128, 4, 0, 1, "tree"),                                # blocks below a request
    (2, [300, 5], [40, 64], 8, 2, 256, 16, 0, 1, "tree"),
    (2, [120], [33], 8, 2, 64, 8, 0, 1, "any"),
    (1, [300, 5], [40, 64], 8, 2, 256, 16, 0, 1, "tree"),
    (1, [120, 31], [33, 1], 8, 2, 128, 1, 0, 1, "tree"),
    (1, [120, 31], [33, 64], 8, 2, 128, 4, 0, 1, "any"),
    (1, [120, 31], [33, 64], 8, 2, 64, 8, 20, 1, "any"),
    (1, [120], [64], 6, 2, 8, 64, 0, 1, "tree"),
    (1, [200, 0], [300, 31], 4, 1, 64, 16, 0, 5, "tree"),
    (0, [200, 0], [300, 31], 4, 1, 64, 16, 0, 5, "tree"),
    (1, list(range(0, 70 * 13, 13)), [1 + i % 5 for i in range(70)], 4, 1, 128, 16, 0, 1, "tree"),   # past 64 sequences
    (2, list(range(0, 130 * 7, 7)), [i % 4 for i in range(130)], 4, 1, 64, 16, 0, 1, "tree"),
    (0, list(range(0, 70 * 5, 5)), [1 + i % 3 for i in range(70)], 2, 1, 32, 16, 0, 1, "chain"),
]


@pytest.mark.parametrize("dtype,ctx,new,H,K,d,bs,window,words,masks", MORE_TREE_CASES)
def test_tree_attention_forms(dtype, ctx, new, H, K, d, bs, window, words, masks):
    """A case for each block of rows, head size and block size that the kernels tell apart, and many sequences."""
    b = Batch(np.random.default_rng(sum(ctx) + d + H + bs), dtype, ctx, new, H, K, d, bs, window, words, masks, spare=1)
    b.check(b.run(_engine()))


@pytest.mark.parametrize("dtype,H,K,d", [(1, 32, 16, 64), (2, 48, 16, 64), (0, 16, 16, 32)])
def test_tree_attention_of_more_items_than_workgroups(dtype, H, K, d):
    """66 sequences, some without rows, of uneven lengths: shares that begin and end inside items, two boundaries in one
    item, and items that no boundary cuts."""
    rng = np.random.default_rng(H + d)
    ctx = [int(x) for x in rng.integers(0, 60, 66)]
    new = [int(x) for x in rng.integers(0, 12, 66)]
    ctx[7], new[7], ctx[60], new[60] = 4000, 9, 2500, 11
    b = Batch(rng, dtype, ctx, new, H, K, d, 16, 0, 1, "tree", spare=1)
    b.check(b.run(_engine()))


@pytest.mark.parametrize("ctx,new,d,bs", [([700, 9], [64, 40], 64, 8), ([700, 9], [64, 40], 128, 4),
                                          ([90], [20], 48, 4), ([90], [20], 64, 2), ([200], [4], 64, 8)])
def test_tree_attention_of_small_e4m3_blocks(ctx, new, d, bs):
    """Blocks that hold 64 pieces of 8 bytes of a head but not of 16, and fewer."""
    b = Batch(np.random.default_rng(d + bs), 2, ctx, new, 8, 2, d, bs, 0, 1, "tree", spare=1)
    b.check(b.run(_engine()))


@pytest.mark.parametrize("dtype,d", [(2, 128), (1, 64), (0, 64)])
def test_tree_attention_of_unaligned_pools(dtype, d):
    """Pools that begin 4 elements inside an allocation (the least that the call takes), and e4m3 half a piece."""
    import torch
    from pagedattentionmetal_amd import PagedAttentionError
    b = Batch(np.random.default_rng(12), dtype, [77, 150], [30, 12], 16, 4, d, 16, 0, 1, "tree")
    host = (b.codes if dtype == 2 else (b.k, b.v))
    ref, vmax, ds = b.exact()
    for shift in (4, 8) if dtype == 2 else (4, 1):
        pools = []
        for x in host:
            flat = torch.zeros(x.size + shift, dtype=to_dev(x).dtype, device="cuda")
            flat[shift:] = to_dev(x).flatten()
            pools.append(flat[shift:].view(x.shape))
        ks, vs = (to_dev(x.view(np.uint16)) for x in b.scales) if dtype == 2 else (None, None)
        q = to_dev(b.q)
        out = torch.zeros_like(q)
        args = (q, *pools, _i32(b.bt), _i32(b.ctx), _i32(b.cu), to_dev(b.mask.view(np.int64)), out, 30,
                _layer(d, 16, 4, 16, dtype))
        if shift == 1:
            with pytest.raises(PagedAttentionError, match="aligned to 4 elements"):
                _engine().tree_attention(*args, k_scale=ks, v_scale=vs)
            continue
        _engine().tree_attention(*args, k_scale=ks, v_scale=vs)
        assert (np.abs(to_host(out).astype(np.float64) - ref) <= b.tolerance(ref, vmax, ds)).all()


@pytest.mark.parametrize("dtype,nodes,bs", [(1, 8, 4), (1, 14, 4), (1, 32, 4), (2, 64, 8), (2, 32, 8)])
def test_tree_attention_of_long_contexts(dtype, nodes, bs):
    """300001 cached tokens of small blocks: a workgroup's share holds more blocks than it keeps the entries of.  A share
    adds at most 300001 / 128 products of two keys to a sum, in f32, one behind the other, and its rounding counts for
    numerator and denominator."""
    import torch
    H, K, d, ctx = 32, 8, 128, 300001
    gen = torch.Generator(device="cuda").manual_seed(nodes)
    L = ctx + nodes
    nb = -(-L // bs)
    G = H // K
    bt = torch.randperm(nb, generator=gen, device="cuda").to(torch.int32).view(1, nb)
    k, v = (torch.randn((nb, bs, K, d), generator=gen, device="cuda", dtype=torch.float16) for _ in range(2))
    scales = None
    pools = (k, v)
    if dtype == 2:
        scales = tuple((x.abs().amax((1, 2, 3)).float() / 448).half() for x in (k, v))
        codes = tuple((x.float() / s.float()[:, None, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                      for x, s in zip((k, v), scales))
        k, v = (c.half() * s[:, None, None, None] for c, s in zip(codes, scales))
        pools = tuple(c.view(torch.uint8) for c in codes)
        scales = tuple(s.view(torch.uint16) for s in scales)
    q = torch.randn((nodes, H, d), generator=gen, device="cuda", dtype=torch.float16)
    on = _paths(_tree(np.random.default_rng(nodes), nodes))
    out = torch.zeros_like(q)
    _engine().tree_attention(q, *pools, bt, _i32([ctx]), _i32([0, nodes]), to_dev(_words(on, 1).view(np.int64)), out,
                             nodes, _layer(d, H, K, bs, dtype), k_scale=scales and scales[0], v_scale=scales and scales[1])
    hidden = torch.zeros((nodes, L), dtype=torch.bool, device="cuda")
    hidden[:, ctx:] = torch.from_numpy(~on).cuda()
    hidden = hidden.repeat_interleave(G, 0)
    for kvh in range(K):
        kk, vv = (x[bt[0].long(), :, kvh].reshape(nb * bs, d)[:L].double() for x in (k, v))
        qh = q[:, kvh * G:(kvh + 1) * G].reshape(-1, d).double()
        x = (qh @ kk.t().contiguous() / d ** 0.5).masked_fill_(hidden, -torch.inf)
        ref = torch.softmax(x, -1) @ vv
        ds = float((qh.abs() @ kk.abs().t().contiguous()).max()) / d ** 0.5
        p = 2 * ((d / 4 + 12) * U * ds + 8 * U) + 2 * (ctx / 128) * U + 2 * HALF
        tol = p * float(vv.abs().max()) + torch.clamp(ref.abs(), min=2.0 ** -14) * HALF
        err = (out[:, kvh * G:(kvh + 1) * G].reshape(-1, d).double() - ref).abs()
        assert bool((err <= tol).all()), (kvh, float((err / tol).max()))


@pytest.mark.parametrize("dtype,d", [(1, 128), (1, 64), (1, 96), (0, 128), (0, 36), (1, 20)])
def test_tree_attention_inf_and_nan_stay_with_the_rows_that_see_them(dtype, d):
    """Inf and NaN of drafted keys and values reach exactly the rows whose masks hold them; those of the cached context,
    before the windows, of blocks no sequence has and behind the last token reach nobody."""
    ctx, new, H, K, bs = [70, 30], [40, 33], 8, 2, 16
    b = Batch(np.random.default_rng(8), dtype, ctx, new, H, K, d, bs, 60, 1, "tree", spare=1)
    k, v = b.k.copy(), b.v.copy()
    used = np.zeros((b.nb, bs), bool)
    for s in range(2):
        for j in range(ctx[s] + new[s]):
            used[b.slot(s, j)] = True
    k[~used] = np.nan
    v[~used] = np.nan
    v[b.slot(0, 2)] = np.inf       # before every row's window
    k[b.slot(0, 3)] = np.nan
    v[b.slot(0, 70 + 9)][1, 3] = np.inf
    v[b.slot(0, 70 + 21)][0, d - 1] = np.nan
    v[b.slot(1, 30 + 4)][0, 0] = -np.inf
    v[b.slot(1, 30 + 4)][0, 1] = np.inf
    got = b.run(_engine(), k=k, v=v).astype(np.float64)
    ref, vmax, ds = b.exact(k=np.nan_to_num(k, nan=0, posinf=0, neginf=0), v=np.nan_to_num(v, nan=0, posinf=0, neginf=0))
    G = H // K
    dirty = np.zeros(got.shape, bool)
    for s, node, kvh, e, val in ((0, 9, 1, 3, np.inf), (0, 21, 0, d - 1, np.nan), (1, 4, 0, 0, -np.inf), (1, 4, 0, 1, np.inf)):
        rows = b.cu[s] + np.flatnonzero(b.visible(s)[:, ctx[s] + node])
        assert len(rows)
        x = got[rows][:, kvh * G:(kvh + 1) * G, e]
        assert (np.isnan(x) if np.isnan(val) else (x == val) | np.isnan(x)).all()
        dirty[np.ix_(rows, range(kvh * G, (kvh + 1) * G), [e])] = True
    err, tol = np.abs(got - ref), b.tolerance(ref, vmax, ds)
    assert (err[~dirty] <= tol[~dirty]).all()


def test_tree_attention_scores_of_the_lowest_values():
    """Keys whose scores are the type's lowest, or -Inf, beside ordinary ones; a row all of whose scores are equal."""
    for dtype in (0, 1):
        b = Batch(np.random.default_rng(4), dtype, [40], [12], 4, 2, 64, 16, 0, 1, "tree")
        k, q = b.k.copy(), b.q.copy()
        q[:, :, 0] = 1.0
        k[b.slot(0, 5)][:, 0] = np.finfo(b.k.dtype).min
        k[b.slot(0, 43)][:, 0] = np.finfo(b.k.dtype).min
        q[3] = 0.0
        got = b.run(_engine(), k=k, q=q)
        k2, (p5, s5), (p43, s43) = k.astype(np.float64), b.slot(0, 5), b.slot(0, 43)
        ref, vmax, ds = b.exact(q=q, k=k2)
        k2[p5, s5], k2[p43, s43] = 0, 0
        ds = b.exact(q=q, k=k2)[2]  # those scores are far below: the others' errors count
        assert (np.abs(got.astype(np.float64) - ref) <= b.tolerance(ref, vmax, ds)).all()


def test_tree_attention_leaves_other_rows_alone():
    """Rows behind the last sequence, and a sequence's rows past max_queries, are left as they were."""
    import torch
    b = Batch(np.random.default_rng(2), 1, [50, 20, 3], [10, 3, 6], 8, 2, 128, 16)
    ref, vmax, ds = b.exact()
    q = np.concatenate([b.q, np.zeros((7, 8, 128), np.float16)])
    b.mask = np.concatenate([b.mask, np.full((7, 1), 3, np.uint64)])
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = b.run(_engine(), out=out, max_queries=6, q=q)
    done = np.r_[0:6, 10:19]
    assert (np.abs(got[done].astype(np.float64) - ref[done]) <= b.tolerance(ref, vmax, ds)[done]).all()
    left = np.r_[6:10, 19:26]
    assert (got[left] == 7).all()


@pytest.mark.parametrize("dtype", [0, 1])
def test_tree_attention_bad_lengths_and_tables_stay_inside(dtype):
    """Lengths past the table, negative ones, row starts out of order and table entries outside the pools change results,
    not memory: the rows of the sound sequence are right."""
    import torch
    b = Batch(np.random.default_rng(6), dtype, [50, 40, 30], [4, 5, 6], 8, 2, 64, 16, spare=1)
    ref, vmax, ds = b.exact()
    b.bt[0] = [1 << 30, -1, 1 << 20, 7, -5][: b.width]
    bad = Batch.__new__(Batch)
    bad.__dict__.update(b.__dict__)
    bad.ctx = [1 << 30, -7, 30]
    got = bad.run(_engine())
    r = slice(b.cu[2], b.cu[3])
    assert (np.abs(got[r].astype(np.float64) - ref[r]) <= b.tolerance(ref, vmax, ds)[r]).all()
    bad.cu = np.array([-4, 1 << 30, 3, 1 << 30], np.int32)
    bad.run(_engine())
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,H,K,d", [(1, 32, 8, 128), (2, 32, 8, 128), (0, 8, 8, 128), (1, 16, 16, 64)])
def test_tree_attention_of_one_node_is_decode(dtype, H, K, d):
    """One drafted token a sequence: the decode of its position, within both results' tolerances."""
    import torch
    ctx = [900, 17, 0, 333]
    b = Batch(np.random.default_rng(5), dtype, ctx, [1] * 4, H, K, d, 16, 0, 1, "tree")
    eng = _engine()
    got = b.run(eng).astype(np.float64)
    out = torch.zeros(b.q.shape, dtype=torch.float32 if dtype == 0 else torch.float16, device="cuda")
    kd, vd = (to_dev(x) for x in (b.codes if dtype == 2 else (b.k, b.v)))
    ks, vs = (to_dev(x.view(np.uint16)) for x in b.scales) if dtype == 2 else (None, None)
    bt = np.where(b.bt < 0, 0, b.bt)
    eng.decode(to_dev(b.q), kd, vd, _i32(bt), _i32([c + 1 for c in ctx]), out, 4, bt.shape[1],
               _layer(d, H, K, 16, dtype), k_scale=ks, v_scale=vs)
    ref, vmax, ds = b.exact()
    assert (np.abs(got - to_host(out)) <= 2 * b.tolerance(ref, vmax, ds)).all()


# ------------------------------------------------------------------ commit


def _commit_ref(b, paths):
    """Pools after the moves, and the lengths."""
    k, v, lens = b.k.copy(), b.v.copy(), []
    for s, path in enumerate(paths):
        n = 0
        for m in path:
            if not (0 <= m < b.new[s]) or (n and m <= path[n - 1]):
                break
            for x in (k, v):
                x[b.slot(s, b.ctx[s] + n)] = x[b.slot(s, b.ctx[s] + m)]
            n += 1
        lens.append(b.ctx[s] + n)
    return k, v, lens


PATHS = [[0, 3, 4, 11, 12, 13, 20, 31, 39], [0], [-1, 2], [2, 5, 5, 6], [0, 1, 2, 3], [1, 0], [3, 40], [0, 7, 1 << 30]]


@pytest.mark.parametrize("dtype,K,d,bs,shift", [(1, 8, 128, 16, 0), (0, 2, 64, 8, 0), (1, 1, 20, 12, 0), (1, 3, 12, 1, 0),
                                                (0, 8, 128, 64, 0), (1, 2, 64, 16, 1)])
def test_tree_commit(dtype, K, d, bs, shift):
    import torch
    n = len(PATHS)
    ctx, new = [37, 0, 5, 16, 15, 90, 3, 8], [40, 1, 9, 12, 4, 2, 40, 30]
    b = Batch(np.random.default_rng(9), dtype, ctx, new, K, K, d, bs)
    paths = np.full((n, 9), -1, np.int32)
    for i, p in enumerate(PATHS):
        paths[i, : len(p)] = p

    def pool(x):  # `shift` elements off its allocation
        flat = torch.zeros(x.size + shift, dtype=to_dev(x[:0]).dtype, device="cuda")
        flat[shift:] = to_dev(x).flatten()
        return flat[shift:].view(x.shape)
    kd, vd, lens = pool(b.k), pool(b.v), _i32(np.zeros(n))
    _engine().tree_commit(kd, vd, _i32(np.where(b.bt < 0, 0, b.bt)), _i32(ctx), _i32(new), _i32(paths),
                          _layer(d, K, K, bs, dtype), new_lengths=lens)
    k, v, ref = _commit_ref(b, PATHS)
    assert to_host(lens).tolist() == ref
    assert np.array_equal(to_host(kd), k) and np.array_equal(to_host(vd), v)


def test_tree_commit_long_paths_and_bad_tables():
    """Paths of more entries than a thread or a wave takes at once; table entries outside the pools move nothing."""
    rng = np.random.default_rng(12)
    b = Batch(rng, 1, [10, 30], [200, 150], 2, 2, 64, 16, words=4)
    paths = np.full((2, 130), -1, np.int32)
    paths[0, :100] = np.sort(rng.permutation(200)[:100])
    paths[1] = np.sort(rng.permutation(150)[:130])
    kd, vd, lens = to_dev(b.k), to_dev(b.v), _i32([0, 0])
    _engine().tree_commit(kd, vd, _i32(np.where(b.bt < 0, 0, b.bt)), _i32(b.ctx), _i32(b.new), _i32(paths),
                          _layer(64, 2, 2, 16, 1), new_lengths=lens)
    k, v, ref = _commit_ref(b, [p[p >= 0].tolist() for p in paths])
    assert to_host(lens).tolist() == ref and np.array_equal(to_host(kd), k) and np.array_equal(to_host(vd), v)
    kd, vd = to_dev(b.k), to_dev(b.v)
    _engine().tree_commit(kd, vd, _i32(np.full(b.bt.shape, 1 << 29)), _i32(b.ctx), _i32(b.new), _i32(paths),
                          _layer(64, 2, 2, 16, 1))
    assert np.array_equal(to_host(kd), b.k) and np.array_equal(to_host(vd), b.v)


@pytest.mark.parametrize("K,d,bs", [(8, 128, 16), (2, 12, 4), (1, 64, 32)])
def test_tree_commit_e4m3_is_an_append_of_the_codes_values(K, d, bs):
    """Codes and scales equal those of appending the accepted tokens' dequantised values at the sequence's end."""
    import torch
    ctx, new = [37, 0, 5, 16], [40, 30, 9, 12]
    paths = np.array([[0, 3, 4, 11, 12, 13, 20, 31, 39], [0, 29, -1, 0, 0, 0, 0, 0, 0], [-1] * 9,
                      [2, 5, 6, 11, 30, 31, 32, 33, 34]], np.int32)
    b = Batch(np.random.default_rng(13), 2, ctx, new, K, K, d, bs)
    b.k[...] *= np.float16(1)
    bt = np.where(b.bt < 0, 0, b.bt)
    eng, lay = _engine(), _layer(d, K, K, bs, 2)
    got = [to_dev(x) for x in b.codes] + [to_dev(x.view(np.int16)) for x in b.scales]
    lens = _i32([0] * 4)
    eng.tree_commit(got[0], got[1], _i32(bt), _i32(ctx), _i32(new), _i32(paths), lay, new_lengths=lens, k_scale=got[2],
                    v_scale=got[3])
    ref = [to_dev(x) for x in b.codes] + [to_dev(x.view(np.int16)) for x in b.scales]
    counts = [9, 2, 0, 4]
    for s in range(4):
        if not counts[s]:
            continue
        at = [b.slot(s, ctx[s] + m) for m in paths[s][: counts[s]]]
        kv = [to_dev(np.stack([x[p, o] for p, o in at])) for x in (b.k, b.v)]
        eng.append_to_cache(kv[0], kv[1], ref[0], ref[1], _i32(bt[s]), ctx[s], counts[s], lay, k_scale=ref[2],
                            v_scale=ref[3])
    assert to_host(lens).tolist() == [c + n for c, n in zip(ctx, counts)]
    for a, r in zip(got, ref):
        assert torch.equal(a, r)


# ------------------------------------------------------------------ together


class Step:
    """A verification step's buffers and calls: plan, norm and rotation into the pools, attention, commit."""

    def __init__(self, rng, dtype, ctx, new, H, K, d, bs, spare_rows=3):
        import torch
        from pagedattentionmetal_amd import RotarySpec
        self.dtype, self.ctx, self.new, self.H, self.K, self.d, self.bs = dtype, ctx, new, H, K, d, bs
        n, rows = len(ctx), sum(new)
        self.cap = rows + spare_rows
        self.layer, self.rotary = _layer(d, H, K, bs, dtype), RotarySpec(d, 10000.0)
        blocks = [-(-(c + t) // bs) for c, t in zip(ctx, new)]
        self.nb, self.width = sum(blocks) + 2, max(blocks)
        t = torch.float32 if dtype == 0 else torch.float16
        z = lambda shape, dt=torch.int32: torch.zeros(shape, dtype=dt, device="cuda")  # noqa: E731
        self.ctx_d, self.new_d = _i32(ctx), _i32(new)
        self.flat, self.parents = z(sum(blocks)), z(self.cap)
        self.paths, self.lens = z((n, 6)), z(n)
        self.plan = dict(cu_queries=z(n + 1), seq_lengths=z(n), block_tables=z((n, self.width)), positions=z(self.cap),
                         slot_mapping=z(self.cap, torch.int64), tree_mask=z((self.cap, 1), torch.int64))
        self.qkv = z((self.cap, (H + 2 * K) * d), t)
        self.q_rot, self.out = z((self.cap, H, d), t), z((self.cap, H, d), t)
        self.kp, self.vp = z((self.nb, bs, K, d), t), z((self.nb, bs, K, d), t)
        self.qw, self.kw = z(d, t), z(d, t)

    def fill(self, seed):
        rng = np.random.default_rng(seed)
        dt, total = NP[self.dtype], self.flat.numel()
        self.flat.copy_(_i32(rng.permutation(self.nb)[:total]))
        self.trees = [_tree(rng, t) for t in self.new]
        par = np.zeros(self.cap, np.int32)
        par[: sum(self.new)] = np.concatenate(self.trees)
        self.parents.copy_(_i32(par))
        paths = np.full(self.paths.shape, -1, np.int32)
        for s, t in enumerate(self.trees):  # a random leaf's path
            node, path = int(rng.integers(0, len(t))), []
            while node >= 0:
                path.insert(0, node)
                node = int(t[node])
            paths[s, : min(6, len(path))] = path[:6]
        self.paths.copy_(_i32(paths))
        self.host_paths = [p[p >= 0].tolist() for p in paths]
        for x, std in ((self.qkv, 1.0), (self.kp, 0.5), (self.vp, 0.5)):
            x.copy_(to_dev((rng.standard_normal(tuple(x.shape)) * std).astype(dt)))
        for x in (self.qw, self.kw):
            x.copy_(to_dev(rng.normal(1, 0.1, self.d).astype(dt)))
        self.out.fill_(7.0)

    def call(self, e):
        H, K, d = self.H, self.K, self.d
        rows = self.qkv
        q, k, v = rows[:, : H * d], rows[:, H * d:(H + K) * d], rows[:, (H + K) * d:]
        e.batch_plan(self.ctx_d, self.new_d, self.flat, self.bs, parents=self.parents, **self.plan)
        e.qk_norm_rope(q.view(-1, H, d), k.view(-1, K, d), self.q_rot, None, self.plan["positions"], self.layer,
                       q_weight=self.qw, k_weight=self.kw, rotary=self.rotary, values=v.view(-1, K, d), k_pool=self.kp,
                       v_pool=self.vp, slot_mapping=self.plan["slot_mapping"])
        e.tree_attention(self.q_rot, self.kp, self.vp, self.plan["block_tables"], self.ctx_d, self.plan["cu_queries"],
                         self.plan["tree_mask"], self.out, max(self.new), self.layer)
        e.tree_commit(self.kp, self.vp, self.plan["block_tables"], self.ctx_d, self.new_d, self.paths, self.layer,
                      new_lengths=self.lens)

    def results(self):
        return [to_host(x).copy() for x in (self.out, self.kp, self.vp, self.lens, self.q_rot[: sum(self.new)])]


@pytest.mark.parametrize("dtype,H,K,d,bs", [(1, 32, 8, 128, 16), (0, 8, 2, 64, 8), (1, 8, 8, 96, 16)])
def test_a_step_is_the_decode_of_the_accepted_path(dtype, H, K, d, bs):
    """Every accepted node's output equals the decode of its position over the committed cache, within twice a row's
    tolerance; rows behind the last sequence keep what they held."""
    import torch
    ctx, new = [100, 0, 37], [12, 5, 20]
    st = Step(np.random.default_rng(1), dtype, ctx, new, H, K, d, bs)
    st.fill(21)
    e = _engine()
    st.call(e)
    out = to_host(st.out).astype(np.float64)
    assert (out[sum(new):] == 7).all()
    cu = to_host(st.plan["cu_queries"])
    assert to_host(st.lens).tolist() == [c + len(p) for c, p in zip(ctx, st.host_paths)]
    dec = torch.empty((1, H, d), dtype=st.out.dtype, device="cuda")
    for s in range(3):
        for depth, node in enumerate(st.host_paths[s]):
            r = int(cu[s]) + node
            assert int(st.plan["positions"][r]) == ctx[s] + depth
            e.decode(st.q_rot[r:r + 1].contiguous(), st.kp, st.vp, st.plan["block_tables"][s:s + 1].contiguous(),
                     _i32([ctx[s] + depth + 1]), dec, 1, st.width, st.layer)
            ref = to_host(dec)[0].astype(np.float64)
            vmax = np.abs(to_host(st.vp).astype(np.float64)).max()
            tol = 2 * ((2 * HALF if dtype else 64 * U) * vmax + 400 * U * vmax) + 2 * _step(dtype, ref)
            assert (np.abs(out[r] - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [1, 0])
def test_a_captured_step_replays(dtype):
    """The step as a HIP graph, replayed over new inputs with eager work between: the eager results bit for bit.  A larger
    call afterwards does not disturb the captured one."""
    import torch
    ctx, new = [300, 20, 1], [16, 9, 30]
    st = Step(np.random.default_rng(1), dtype, ctx, new, 16, 4, 64, 16)
    e = _engine()
    e.synchronous = False
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        e.set_stream(stream)
        want = []
        for seed in (31, 32, 33):
            st.fill(seed)
            st.call(e)
            stream.synchronize()
            want.append(st.results())
        graph = torch.cuda.CUDAGraph()
        st.fill(34)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            e.set_stream(torch.cuda.current_stream())
            st.call(e)
        big = Batch(np.random.default_rng(3), dtype, [5000, 4000], [60, 64], 16, 4, 64, 16)
        for n, seed in enumerate((31, 32, 33, 31)):
            st.fill(seed)
            graph.replay()
            stream.synchronize()
            for a, b in zip(st.results(), want[n % 3]):
                assert np.array_equal(a, b)
            big.run(e)  # a larger workspace between the replays
    e.set_stream(None)
    e.synchronize()


def test_a_captured_call_that_would_wait_is_refused():
    import torch
    st = Step(np.random.default_rng(1), 1, [30], [4], 8, 2, 64, 16)
    st.fill(3)
    e = _engine()
    from pagedattentionmetal_amd import PagedAttentionError
    stream = torch.cuda.Stream()
    e.set_stream(stream)
    torch.cuda.synchronize()
    st.call(e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        with pytest.raises(PagedAttentionError, match="asynchronous"):
            st.call(e)
        st.out.zero_()
    graph.replay()
    stream.synchronize()
    assert (to_host(st.out) == 0).all()


def test_two_engines_on_two_streams():
    """Two contexts at once on streams of their own: each has its workspace."""
    import torch
    steps, engines, streams, want = [], [], [], []
    for i in range(2):
        st = Step(np.random.default_rng(1), 1, [900 + i, 40], [16, 30], 16, 4, 128, 16)
        st.fill(50 + i)
        st.call(_engine())
        want.append(st.results())
        e = _engine()
        e.synchronous = False
        s = torch.cuda.Stream()
        e.set_stream(s)
        steps.append(st), engines.append(e), streams.append(s)
    for _ in range(5):
        for st, i in zip(steps, (50, 51)):
            st.fill(i)
        torch.cuda.synchronize()
        for st, e in zip(steps, engines):
            st.call(e)
        for e in engines:
            e.synchronize()
        for st, w in zip(steps, want):
            for a, b in zip(st.results(), w):
                assert np.array_equal(a, b)


def test_strict_code_object_and_injected_failures():
    from pagedattentionmetal_amd import PagedAttentionError
    st = Step(np.random.default_rng(1), 1, [30], [4], 8, 2, 64, 16)
    st.fill(3)
    e = _engine()
    st.call(e)
    want = st.results()
    st.fill(3)
    e.debug_fail_next_launches(1)  # retried: nothing was enqueued
    st.call(e)
    assert all(np.array_equal(a, b) for a, b in zip(st.results(), want))
    e.load_module()
    st.fill(3)
    st.call(e)  # from the library
    assert all(np.array_equal(a, b) for a, b in zip(st.results(), want))
    e.set_module_strict(True)
    with pytest.raises(PagedAttentionError, match="not in the code object"):
        st.call(e)


def test_empty_masks_and_parents_are_refused():
    """A mask of no words and parents of no entries have no address, which elsewhere says that there are none."""
    import torch
    from pagedattentionmetal_amd import PagedAttentionError
    eng = _engine()
    i32, i64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")
    q = torch.zeros(2, 8, 64, dtype=torch.float16, device="cuda")
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(PagedAttentionError, match="tree_mask needs one row"):
        eng.tree_attention(q, pool, pool, torch.zeros(1, 4, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32),
                           torch.zeros(2, 0, **i64), torch.empty_like(q), 2, _layer(64, 8, 2))
    with pytest.raises(PagedAttentionError, match="buffer of its own"):
        eng.tree_attention(q, pool, pool, torch.zeros(1, 4, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32),
                           torch.zeros(2, 1, **i64), q, 2, _layer(64, 8, 2))
    one = torch.zeros(1, **i32)
    out = dict(cu_queries=torch.zeros(2, **i32), seq_lengths=torch.zeros(1, **i32), block_tables=torch.zeros(1, 4, **i32),
               positions=torch.zeros(2, **i32), slot_mapping=torch.zeros(2, **i64))
    with pytest.raises(PagedAttentionError, match="parents needs one entry"):
        eng.batch_plan(one, one, one, 16, **out, parents=torch.zeros(0, **i32))
    with pytest.raises(PagedAttentionError, match="tree_mask needs one row"):
        eng.batch_plan(one, one, one, 16, **out, tree_mask=torch.zeros(2, 0, **i64))
