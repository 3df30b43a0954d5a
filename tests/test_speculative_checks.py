"""The speculative-decoding calls' refusals and host arithmetic, without a GPU: every request is checked before
the device is touched, so the pointers here are never read."""
import ctypes as C
import math

import pytest

from pagedattentionmetal_amd import PagedAttentionEngine, PagedAttentionError, PagedLayerSpec, RotarySpec, _lib

FAKE = 1 << 20  # an aligned address
LAYER = dict(head_dim=64, num_heads=8, num_kv_heads=2, block_size=16, data_type=1, window_size=0)


def _layer(**kw):
    return _lib.LayerSpec(*[{**LAYER, **kw}[f] for f, _ in _lib.LayerSpec._fields_])


def _request(cls, base, **kw):
    r = cls()
    for f, v in {**base, **kw}.items():
        setattr(r, f, v)
    return r


def _refused(name, r, text):
    e = PagedAttentionEngine()
    lib = _lib.load()
    assert getattr(lib, "pam_engine_" + name)(e.handle, C.byref(r)) == -1
    msg = lib.pam_last_error(e.handle).decode()
    assert text in msg, msg


PLAN = dict(context_lens=FAKE, query_lens=FAKE, block_list=FAKE, block_list_len=10, num_seqs=2, block_size=16,
            max_num_blocks=8, max_rows=4, cu_queries=FAKE, seq_lengths=FAKE, block_tables=FAKE, positions=FAKE,
            slot_mapping=FAKE)


@pytest.mark.parametrize("change,text", [
    (dict(num_seqs=0), "numSeqs must be positive"), (dict(block_size=0), "blockSize must be positive"),
    (dict(max_num_blocks=-1), "maxNumBlocks must be positive"), (dict(max_rows=0), "maxRows must be positive"),
    (dict(max_num_blocks=1 << 30), "2^31 - 1 tokens"), (dict(block_list_len=-1), "must not be negative"),
    (dict(tree_mask=FAKE, mask_words=0), "maskWords must be 1 to 16"),
    (dict(tree_mask=FAKE, mask_words=17), "maskWords must be 1 to 16"),
    (dict(slot_mapping=None), "null buffer"), (dict(block_list=None), "null buffer"),
])
def test_batch_plan_refusals(change, text):
    _refused("batch_plan", _request(_lib.BatchPlanRequest, PLAN, **change), text)


def _norm(**kw):
    rotary = kw.pop("rotary", (64, 0, 10000.0))
    lay = kw.pop("layer", {})
    base = dict(q=FAKE, k=FAKE, q_out=FAKE + 4096, k_out=FAKE + 8192, positions=FAKE, num_tokens=4, eps=1e-6,
                normalize=True, layer=_layer(**lay), rotary=_lib.RotarySpecC(*rotary, None))
    return _request(_lib.QkNormRopeRequest, base, **kw)


POOL = dict(values=FAKE, k_pool=FAKE, v_pool=FAKE, slot_mapping=FAKE)


@pytest.mark.parametrize("change,text", [
    (dict(num_tokens=0), "numTokens must be positive"), (dict(layer=dict(head_dim=66)), "multiple of 4"),
    (dict(layer=dict(head_dim=260)), "at most 256"), (dict(layer=dict(num_heads=7)), "divisible"),
    (dict(rotary=(63, 0, 1e4)), "rotaryDim"), (dict(rotary=(66, 0, 1e4)), "rotaryDim"),
    (dict(rotary=(-2, 0, 1e4)), "rotaryDim"), (dict(rotary=(64, 0, 0.0)), "base must be positive"),
    (dict(rotary=(64, 0, math.inf)), "base must be positive"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
    (dict(positions=None), "needs positions"), (dict(rotary=(0, 0, 0.0), normalize=False), "neither norm nor rotation"),
    (dict(normalize=False, q_weight=FAKE), "weights go with the norm"), (dict(q=None), "null buffer"),
    (dict(k_out=None), "null buffer"), (dict(q_stride=511), "rows overlap"), (dict(k_stride=-128), "rows overlap"),
    (dict(k_pool=FAKE), "go together"), ({**POOL, "values": None}, "go together"),
    ({**POOL, "layer": dict(data_type=2)}, "FP8 pools"), (dict(q_bytes=4 * 512 * 2 - 1), "Q buffer is too small"),
    (dict(q_stride=1024, q_bytes=(3 * 1024 + 512) * 2 - 2), "Q buffer is too small"),
    (dict(positions_bytes=15), "positions buffer is too small"),
    ({**POOL, "slot_mapping_bytes": 31}, "slotMapping buffer is too small"),
    ({**POOL, "k_pool_bytes": 100, "v_pool_bytes": 1 << 20}, "K pool buffer is too small"),
    (dict(q_out=FAKE, q_stride=1024), "in place has Q's stride"),
])
def test_qk_norm_rope_refusals(change, text):
    _refused("qk_norm_rope", _norm(**change), text)


def test_qk_norm_rope_backward_refusals():
    base = dict(q=FAKE, k=FAKE, d_q_out=FAKE + 64, d_k_out=FAKE + 64, d_q=FAKE + 128, d_k=FAKE + 128, positions=FAKE,
                num_tokens=4, eps=1e-6, normalize=True, layer=_layer(), rotary=_lib.RotarySpecC(64, 0, 1e4, None))
    for change, text in [(dict(num_tokens=-1), "numTokens"), (dict(d_q=None), "null buffer"),
                         (dict(d_q=FAKE), "buffers of their own"), (dict(d_q_stride=100), "rows overlap"),
                         (dict(d_k_bytes=8), "K gradient buffer is too small"),
                         (dict(normalize=False, d_q_weight=FAKE), "weights go with the norm"),
                         (dict(d_q=FAKE + 64), "buffers of their own")]:
        _refused("qk_norm_rope_backward", _request(_lib.QkNormRopeBackwardRequest, base, **change), text)


def _tree(**kw):
    lay = kw.pop("layer", {})
    base = dict(q=FAKE, output=FAKE, k_pool=FAKE, v_pool=FAKE, block_tables=FAKE, context_lens=FAKE, cu_queries=FAKE,
                tree_mask=FAKE, mask_words=1, num_seqs=2, max_num_blocks=8, max_queries=64, total_rows=100,
                layer=_layer(**lay), k_pool_bytes=1 << 20, v_pool_bytes=1 << 20)
    return _request(_lib.TreeAttentionRequest, base, **kw)


@pytest.mark.parametrize("change,text", [
    (dict(num_seqs=0), "numSeqs"), (dict(max_num_blocks=0), "maxNumBlocks"), (dict(max_queries=0), "maxQueries must"),
    (dict(total_rows=0), "totalRows"), (dict(num_seqs=65536), "at most 65535"),
    (dict(max_queries=65), "tree mask's bits"), (dict(mask_words=0), "tree mask's bits"),
    (dict(max_num_blocks=1 << 27), "2^31 - 4096 tokens"), (dict(q=None), "null buffer"),
    (dict(layer=dict(data_type=2)), "FP8 tree attention needs"), (dict(layer=dict(window_size=-1)), "windowSize"),
    (dict(k_pool_bytes=0), "sizes are needed"), (dict(v_pool_bytes=100), "K pool buffer is too small"),
    (dict(q_bytes=1000), "Q buffer is too small"), (dict(output_bytes=1000), "output buffer is too small"),
    (dict(tree_mask_bytes=799), "treeMask buffer is too small"), (dict(cu_queries_bytes=8), "cuQueries"),
    (dict(context_lens_bytes=4), "contextLens"), (dict(block_tables_bytes=60), "blockTables"),
    (dict(q=FAKE + 2), "aligned to 4 elements"), (dict(k_pool=FAKE + 4), "aligned to 4 elements"),
    (dict(layer=dict(head_dim=50)), "multiple of 4"),
])
def test_tree_attention_refusals(change, text):
    _refused("tree_attention", _tree(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(num_seqs=0), "numSeqs"), (dict(max_path=0), "maxPath"), (dict(paths=None), "null buffer"),
    (dict(new_lengths=FAKE), "buffer of its own"), (dict(layer=_layer(data_type=2)), "FP8 tree commit needs"),
    (dict(k_pool_bytes=0), "sizes are needed"), (dict(paths_bytes=60), "paths buffer is too small"),
    (dict(query_lens_bytes=4), "queryLens"), (dict(k_pool=FAKE + 1), "aligned"),
])
def test_tree_commit_refusals(change, text):
    base = dict(k_pool=FAKE, v_pool=FAKE, block_tables=FAKE, context_lens=FAKE, query_lens=FAKE, paths=FAKE,
                num_seqs=2, max_num_blocks=8, max_path=8, layer=_layer(), k_pool_bytes=1 << 20, v_pool_bytes=1 << 20)
    _refused("tree_commit", _request(_lib.TreeCommitRequest, base, **change), text)


def test_a_null_request_or_context_is_refused():
    lib = _lib.load()
    e = PagedAttentionEngine()
    for name in ("batch_plan", "qk_norm_rope", "qk_norm_rope_backward", "tree_attention", "tree_commit"):
        assert getattr(lib, "pam_engine_" + name)(e.handle, None) == -1
    assert lib.pam_engine_tree_attention(None, C.byref(_tree())) == -1
    assert lib.pam_context_device(None) == -1 and lib.pam_context_device(e.handle) == -1


def test_rotary_spec():
    r = RotarySpec(8, 100.0)
    assert r.inv_freq == [100.0 ** (-i / 4) for i in range(4)]
    assert RotarySpec(4, inv_freq=[1.0, 0.25]).inv_freq == [1.0, 0.25]
    assert RotarySpec(0).inv_freq == []
    for bad in (dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=4, base=0.0), dict(rotary_dim=4, base=math.nan),
                dict(rotary_dim=4, inv_freq=[1.0]), dict(rotary_dim=4, inv_freq=[1.0, math.inf])):
        with pytest.raises(PagedAttentionError):
            RotarySpec(**bad)


@pytest.mark.parametrize("cls", [_lib.BatchPlanRequest, _lib.QkNormRopeRequest, _lib.QkNormRopeBackwardRequest,
                                 _lib.TreeAttentionRequest, _lib.TreeCommitRequest])
def test_packed_requests_are_the_structs_bytes(cls):
    """Every field of its own value, packed and through the ctypes structure."""
    values, r, n = [], cls(), 0

    def fill(s):
        nonlocal n
        for name, t in s._fields_:
            if issubclass(t, C.Structure):
                fill(getattr(s, name))
                continue
            n += 1
            v = True if t is C.c_bool else (n * 0.5 if t in (C.c_float, C.c_double) else n * 1000003)
            setattr(s, name, v)
            values.append(v)
    fill(r)
    got, ref = _lib.packer(cls)(*values), bytes(r)
    assert len(got) == C.sizeof(cls)
    back = cls.from_buffer_copy(got)

    def same(a, b):
        for name, t in a._fields_:
            x, y = getattr(a, name), getattr(b, name)
            assert same(x, y) if issubclass(t, C.Structure) else x == y, name
        return True
    assert same(r, back) and len(ref) == len(got)


def test_host_tensors_and_wrong_types_are_refused():
    import torch
    e = PagedAttentionEngine()
    lay = PagedLayerSpec(64, 8, 2, 16, 1)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(PagedAttentionError, match="not on a GPU"):
        e.batch_plan(i, i, i, 16, torch.zeros(3, dtype=torch.int32), i, i.view(2, 1), i, torch.zeros(2, dtype=torch.int64))
    x = torch.zeros(2, 8, 64, dtype=torch.float16)
    with pytest.raises(PagedAttentionError, match="not on a GPU"):
        e.qk_norm_rope(x, x[:, :2], x, x[:, :2], None, lay)
    with pytest.raises(PagedAttentionError, match="not on a GPU"):
        e.tree_attention(x, x, x, i.view(2, 1), i, i, None, x, 1, lay)
    with pytest.raises(PagedAttentionError, match="not on a GPU"):
        e.tree_commit(x, x, i.view(2, 1), i, i, i.view(2, 1), lay)


BIG = (1 << 31) - 1


@pytest.mark.parametrize("change,text", [
    (dict(), "the output needs a buffer of its own"),
    (dict(output=FAKE + 4096, layer=dict(num_heads=1 << 17, num_kv_heads=1 << 16)), "at most 65535 key heads"),
    (dict(layer=dict(num_heads=BIG // 2, num_kv_heads=1), total_rows=BIG, max_queries=64, num_seqs=1,
          mask_words=1), "overflow"),
    (dict(mask_words=BIG, total_rows=BIG), "overflow"),
])
def test_tree_attention_refuses_aliases_and_sizes_past_64_bits(change, text):
    _refused("tree_attention", _tree(**change), text)


def test_sizes_past_64_bits_are_refused():
    """A block of 2^64 bytes, whose count of bytes wraps to zero, and rows whose ends do not fit."""
    lay = _layer(block_size=1 << 30, num_heads=1 << 24, num_kv_heads=1 << 24, head_dim=256, data_type=0)
    base = dict(k_pool=FAKE, v_pool=FAKE, block_tables=FAKE, context_lens=FAKE, query_lens=FAKE, paths=FAKE,
                num_seqs=2, max_num_blocks=1, max_path=8, layer=lay, k_pool_bytes=1 << 20, v_pool_bytes=1 << 20)
    _refused("tree_commit", _request(_lib.TreeCommitRequest, base), "overflow")
    base.update(layer=_layer(block_size=1), num_seqs=BIG, max_num_blocks=BIG)
    _refused("tree_commit", _request(_lib.TreeCommitRequest, base), "overflow")
    _refused("qk_norm_rope", _norm(num_tokens=BIG, q_stride=1 << 40), "overflow")
    _refused("qk_norm_rope", _norm(num_tokens=1, k_out_stride=(1 << 62) + 1), "overflow")
