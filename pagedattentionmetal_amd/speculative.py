"""The engine's speculative-decoding calls (no reference counterpart): batch plans, norm and rotation of query and
key heads with their gradients, attention of drafted trees and commits of accepted paths.

The calls take torch device tensors, check them here (type, shape, device, contiguity) and pass the request as packed
bytes: a verification step makes four of them a layer, each a few microseconds of GPU work.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib
from .errors import PagedAttentionError

_BAD = "Invalid paged attention configuration: "


def _want(ok, message):
    if not ok:
        raise PagedAttentionError(_BAD + message)


class RotarySpec:
    """The position rotation of query and key heads: the first ``rotary_dim`` dims of a head (even) turn by
    position * inv_freq[i], pair i being dims (i, i + rotary_dim / 2) or, ``interleaved``, (2i, 2i + 1).
    ``inv_freq`` (rotary_dim / 2 numbers) replaces base^(-2i / rotary_dim)."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, inv_freq=None):
        rotary_dim = int(rotary_dim)
        if rotary_dim < 0 or rotary_dim % 2:
            raise PagedAttentionError("Invalid paged attention configuration: rotaryDim must be even and at most "
                                      "headDim.")
        if inv_freq is None:
            if not (math.isfinite(base) and base > 0):
                raise PagedAttentionError("Invalid paged attention configuration: the rotation's base must be "
                                          "positive.")
            inv_freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        freq = [float(f) for f in inv_freq]
        if len(freq) != rotary_dim // 2 or not all(math.isfinite(f) for f in freq):
            raise PagedAttentionError("Invalid paged attention configuration: inv_freq needs rotary_dim / 2 finite "
                                      "numbers.")
        self.rotary_dim, self.base, self.interleaved, self.inv_freq = rotary_dim, float(base), bool(interleaved), freq
        self._freq = (C.c_double * max(1, len(freq)))(*freq)
        # the fields of pam_rotary_spec
        self._fields = (rotary_dim, int(self.interleaved), self.base, C.addressof(self._freq))


class _Calls:
    """What the calls need once: torch's types, the packers and the library's functions."""

    def __init__(self):
        import torch
        self.i32, self.i64, self.f32, self.f16, self.u8 = (torch.int32, torch.int64, torch.float32, torch.float16,
                                                           torch.uint8)
        self.current_device = torch.cuda.current_device
        for name, cls in (("batch_plan", _lib.BatchPlanRequest), ("qk_norm_rope", _lib.QkNormRopeRequest),
                          ("qk_norm_rope_backward", _lib.QkNormRopeBackwardRequest),
                          ("tree_attention", _lib.TreeAttentionRequest), ("tree_commit", _lib.TreeCommitRequest)):
            setattr(self, "pack_" + name, _lib.packer(cls))
            setattr(self, name, _lib.raw("pam_engine_" + name))


_calls = None


def _c() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


def _ptr(t, dtype, dev, name):
    """A device buffer's address: contiguous, of its type, on GPU `dev`; 0 for None."""
    if t is None:
        return 0
    if t.get_device() != dev or t.dtype is not dtype or not t.is_contiguous():
        if not t.is_cuda:
            raise PagedAttentionError(_BAD + f"{name} is not on a GPU.")
        if t.get_device() != dev:
            raise PagedAttentionError(_BAD + f"{name} is on another GPU.")
        if t.dtype is not dtype:
            raise PagedAttentionError(_BAD + f"{name} is {t.dtype}, expected {dtype}.")
        raise PagedAttentionError("buffers must be contiguous")
    return t.data_ptr()


def _rows(t, dtype, dev, shape, name):
    """A [tokens, heads, head_dim] tensor whose heads are contiguous: its address and row stride."""
    n, heads, d = shape
    s = t.stride()
    if (t.get_device() != dev or t.dtype is not dtype or t.shape != shape or s[2] != 1 or
            (s[1] != d and heads != 1) or (s[0] < heads * d and n > 1)):
        _want(t.is_cuda, f"{name} is not on a GPU.")
        _want(t.get_device() == dev, f"{name} is on another GPU.")
        _want(t.dtype is dtype, f"{name} is {t.dtype}, expected {dtype}.")
        _want(t.shape == shape, f"{name} is {list(t.shape)}, expected {list(shape)}.")
        _want(False, f"{name}'s heads must be contiguous.")
    return t.data_ptr(), (s[0] if n > 1 else heads * d)


def _layer(layer):
    return (layer.head_dim, layer.num_heads, layer.num_kv_heads, layer.block_size, int(layer.data_type),
            layer.window_size)


_NO_ROTATION = (0, 0, 1.0, 0)


class SpeculativeCalls:
    """The calls, as methods of PagedAttentionEngine."""

    _gpu = -1  # the context's GPU, once it has one

    def _on(self, t, name):
        """The GPU of the call's first buffer, which is the engine's."""
        dev = t.get_device()
        if dev < 0:
            raise PagedAttentionError(_BAD + f"{name} is not on a GPU.")
        if dev != self._gpu:
            have = _lib.load().pam_context_device(self._ctx)
            if have < 0:  # the context takes the current GPU
                have = _c().current_device()
            _want(have == dev, f"{name} is on GPU {dev}, the engine on {have}.")
            self._gpu = dev
        return dev

    def batch_plan(self, context_lens, query_lens, block_list, block_size, cu_queries, seq_lengths, block_tables,
                   positions, slot_mapping, parents=None, tree_mask=None, status=None):
        """Block tables, slot maps, positions and tree masks of a ragged batch, built on the GPU from its lengths
        (pam_engine_batch_plan).  int32 device tensors, slot_mapping and tree_mask int64; all but status are
        written whole: block_tables [sequences, width], positions and slot_mapping [rows at most], tree_mask
        [rows at most, words].  ``parents``: each row's parent among its sequence's new tokens, -1 for none."""
        c = _c()
        dev, i32 = self._on(context_lens, "context_lens"), c.i32
        n, rows, width, words = context_lens.numel(), positions.numel(), block_tables.shape, 0
        if query_lens.numel() != n or cu_queries.numel() != n + 1 or seq_lengths.numel() != n:
            _want(False, f"the lengths of {n} sequences do not match.")
        _want(len(width) == 2 and width[0] == n, "block_tables needs one row per sequence.")
        _want(slot_mapping.numel() == rows, "positions and slot_mapping need the same rows.")
        if tree_mask is not None:
            words = tree_mask.shape[1] if tree_mask.dim() == 2 else 0
            _want(words > 0 and tree_mask.shape[0] == rows, "tree_mask needs one row per position.")
        if parents is not None and parents.numel() == 0:
            _want(False, "parents needs one entry per new token.")
        r = c.pack_batch_plan(
            _ptr(context_lens, i32, dev, "context_lens"), _ptr(query_lens, i32, dev, "query_lens"),
            _ptr(block_list, i32, dev, "block_list"), _ptr(parents, i32, dev, "parents"), block_list.numel(),
            0 if parents is None else parents.numel(), n, block_size, width[1], rows, words,
            _ptr(cu_queries, i32, dev, "cu_queries"), _ptr(seq_lengths, i32, dev, "seq_lengths"),
            _ptr(block_tables, i32, dev, "block_tables"), _ptr(positions, i32, dev, "positions"),
            _ptr(slot_mapping, c.i64, dev, "slot_mapping"), _ptr(tree_mask, c.i64, dev, "tree_mask"),
            _ptr(status, i32, dev, "status"))
        if c.batch_plan(self._ctx, r):
            self._check(-1)

    def qk_norm_rope(self, q, k, q_out, k_out, positions, layer, q_weight=None, k_weight=None, eps: float = 1e-6,
                     rotary: RotarySpec = None, normalize: bool = True, values=None, k_pool=None, v_pool=None,
                     slot_mapping=None):
        """RMS norm of every query and key head and the rotation to its token's position in one pass
        (pam_engine_qk_norm_rope).  q, k, values and the outputs are [tokens, heads, head_dim] of any row stride;
        q_out may be q, k_out k.  With the pools and an int64 slot_mapping the keys and values go to their slots
        too, and k_out may be None."""
        c = _c()
        dev = self._on(q, "q")
        io = c.f32 if layer.data_type == 0 else c.f16
        n, d = q.shape[0], layer.head_dim
        qs, ks = (n, layer.num_heads, d), (n, layer.num_kv_heads, d)
        self._norm_sizes(n, d, positions, q_weight, k_weight)
        qp, q_stride = _rows(q, io, dev, qs, "q")
        kp, k_stride = _rows(k, io, dev, ks, "k")
        qo, qo_stride = _rows(q_out, io, dev, qs, "q_out")
        ko, ko_stride = (0, 0) if k_out is None else _rows(k_out, io, dev, ks, "k_out")
        vp = v_stride = k_bytes = v_bytes = 0
        if values is not None:
            vp, v_stride = _rows(values, io, dev, ks, "values")
        if k_pool is not None and v_pool is not None:
            k_bytes, v_bytes = k_pool.numel() * k_pool.element_size(), v_pool.numel() * v_pool.element_size()
        _want(slot_mapping is None or slot_mapping.numel() == n, "slot_mapping needs one entry per token.")
        r = c.pack_qk_norm_rope(
            qp, kp, qo, ko, _ptr(q_weight, io, dev, "q_weight"), _ptr(k_weight, io, dev, "k_weight"),
            _ptr(positions, c.i32, dev, "positions"), q_stride, k_stride, qo_stride, ko_stride, n, *_layer(layer),
            *(_NO_ROTATION if rotary is None else rotary._fields), eps, normalize, vp, v_stride,
            _ptr(k_pool, io, dev, "k_pool"), _ptr(v_pool, io, dev, "v_pool"),
            _ptr(slot_mapping, c.i64, dev, "slot_mapping"), 0, 0, 0, 0, 0, 0, k_bytes, v_bytes, 0)
        if c.qk_norm_rope(self._ctx, r):
            self._check(-1)

    @staticmethod
    def _norm_sizes(n, d, positions, *weights):
        _want(positions is None or positions.numel() == n, "positions need one entry per token.")
        for w in weights:
            _want(w is None or w.numel() == d, "weights have head_dim entries.")

    def qk_norm_rope_backward(self, q, k, d_q_out, d_k_out, d_q, d_k, positions, layer, q_weight=None, k_weight=None,
                              d_q_weight=None, d_k_weight=None, eps: float = 1e-6, rotary: RotarySpec = None,
                              normalize: bool = True):
        """Gradients of qk_norm_rope's outputs: d_q, d_k and the weights' (float32), all written
        (pam_engine_qk_norm_rope_backward).  q and k are the forward's inputs."""
        c = _c()
        dev = self._on(q, "q")
        io = c.f32 if layer.data_type == 0 else c.f16
        n, d = q.shape[0], layer.head_dim
        qs, ks = (n, layer.num_heads, d), (n, layer.num_kv_heads, d)
        self._norm_sizes(n, d, positions, q_weight, k_weight, d_q_weight, d_k_weight)
        qp, q_stride = _rows(q, io, dev, qs, "q")
        kp, k_stride = _rows(k, io, dev, ks, "k")
        gq, gq_stride = _rows(d_q_out, io, dev, qs, "d_q_out")
        gk, gk_stride = _rows(d_k_out, io, dev, ks, "d_k_out")
        dq, dq_stride = _rows(d_q, io, dev, qs, "d_q")
        dk, dk_stride = _rows(d_k, io, dev, ks, "d_k")
        r = c.pack_qk_norm_rope_backward(
            qp, kp, gq, gk, dq, dk, _ptr(q_weight, io, dev, "q_weight"), _ptr(k_weight, io, dev, "k_weight"),
            _ptr(d_q_weight, c.f32, dev, "d_q_weight"), _ptr(d_k_weight, c.f32, dev, "d_k_weight"),
            _ptr(positions, c.i32, dev, "positions"), q_stride, k_stride, gq_stride, gk_stride, dq_stride, dk_stride, n,
            *_layer(layer), *(_NO_ROTATION if rotary is None else rotary._fields), eps, normalize, 0, 0, 0, 0, 0, 0, 0)
        if c.qk_norm_rope_backward(self._ctx, r):
            self._check(-1)

    def _pools(self, c, layer, dev, k_pool, v_pool, k_scale, v_scale):
        """Addresses and sizes of the pools and their scales."""
        t = c.f16 if layer.data_type == 1 else (c.f32 if layer.data_type == 0 else c.u8)
        kb = k_pool.numel() * k_pool.element_size()
        vb = v_pool.numel() * v_pool.element_size()
        ks = vs = 0
        if layer.data_type == 2:
            _want(k_scale is not None and v_scale is not None, "FP8 pools need the K and V scale pools.")
            blocks = min(kb, vb) // max(1, layer.block_size * layer.num_kv_heads * layer.head_dim)
            for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if s.element_size() != 2 or s.numel() < blocks:
                    _want(False, f"{name} needs one half per block.")
            ks = _ptr(k_scale, k_scale.dtype, dev, "k_scale")
            vs = _ptr(v_scale, v_scale.dtype, dev, "v_scale")
        return _ptr(k_pool, t, dev, "k_pool"), _ptr(v_pool, t, dev, "v_pool"), ks, vs, kb, vb

    def tree_attention(self, q, k_pool, v_pool, block_tables, context_lens, cu_queries, tree_mask, output,
                       max_queries, layer, k_scale=None, v_scale=None):
        """Attention of drafted trees over the cache (pam_engine_tree_attention): q and output [rows, heads,
        head_dim], sequence s's rows cu_queries[s] .. cu_queries[s + 1] - 1 (at most max_queries), its drafted keys
        and values in the pools from position context_lens[s] on.  tree_mask [rows, words] int64, or None for
        chains."""
        c = _c()
        dev = self._on(q, "q")
        io, i32 = c.f32 if layer.data_type == 0 else c.f16, c.i32
        n, shape, table, words = context_lens.numel(), q.shape, block_tables.shape, 0
        if not (len(shape) == 3 and shape[1] == layer.num_heads and shape[2] == layer.head_dim and
                output.shape == shape):
            _want(False, f"q and output are [rows, {layer.num_heads}, {layer.head_dim}].")
        _want(len(table) == 2 and table[0] == n and cu_queries.numel() == n + 1,
              "block_tables and cu_queries need the sequences of context_lens.")
        if tree_mask is not None:
            words = tree_mask.shape[1] if tree_mask.dim() == 2 else 0
            _want(words > 0 and tree_mask.shape[0] == shape[0], "tree_mask needs one row per query row.")
        kp, vp, ks, vs, kb, vb = self._pools(c, layer, dev, k_pool, v_pool, k_scale, v_scale)
        r = c.pack_tree_attention(
            _ptr(q, io, dev, "q"), _ptr(output, io, dev, "output"), kp, vp, _ptr(block_tables, i32, dev, "block_tables"),
            _ptr(context_lens, i32, dev, "context_lens"), _ptr(cu_queries, i32, dev, "cu_queries"),
            _ptr(tree_mask, c.i64, dev, "tree_mask"), words, n, table[1], max_queries, shape[0], *_layer(layer), ks, vs,
            0, 0, kb, vb, 0, 0, 0, 0)
        if c.tree_attention(self._ctx, r):
            self._check(-1)

    def tree_commit(self, k_pool, v_pool, block_tables, context_lens, query_lens, paths, layer, new_lengths=None,
                    k_scale=None, v_scale=None):
        """The accepted path of every sequence moved to the end of its cached tokens (pam_engine_tree_commit):
        paths [sequences, at most] int32, a path's nodes in rising order, -1 behind them."""
        c = _c()
        dev, i32 = self._on(context_lens, "context_lens"), c.i32
        n, table, path = context_lens.numel(), block_tables.shape, paths.shape
        _want(len(table) == 2 and table[0] == n and len(path) == 2 and path[0] == n and query_lens.numel() == n and
              (new_lengths is None or new_lengths.numel() == n),
              "every argument needs the sequences of context_lens.")
        kp, vp, ks, vs, kb, vb = self._pools(c, layer, dev, k_pool, v_pool, k_scale, v_scale)
        r = c.pack_tree_commit(
            kp, vp, ks, vs, _ptr(block_tables, i32, dev, "block_tables"), _ptr(context_lens, i32, dev, "context_lens"),
            _ptr(query_lens, i32, dev, "query_lens"), _ptr(paths, i32, dev, "paths"),
            _ptr(new_lengths, i32, dev, "new_lengths"), n, table[1], path[1], *_layer(layer), kb, vb, 0, 0, 0, 0)
        if c.tree_commit(self._ctx, r):
            self._check(-1)
