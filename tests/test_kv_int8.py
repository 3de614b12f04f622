"""Refusals of the INT8 key/value cache's calls: everything is checked before a device is touched."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def sgq():
    from __graft_entry__ import load_package
    return load_package()


ONE, TWO, ODD = C.c_void_p(256), C.c_void_p(1 << 20), C.c_void_p(260)      # never dereferenced: validation comes first


def cache(sgq, batch=2, kv=2, max_seq=16, dim=128, k=256, ks=256, v=256, vs=256):
    return C.byref(sgq.CacheInt8(k, ks, v, vs, batch, kv, max_seq, dim))


def store(sgq, c, qkv=ONE, stride=1024, t=1, heads=4, cos=ONE, sin=ONE, rows=16, pos=ONE, ps=1, n_new=None, offset=None, q=TWO, qs=512):
    return sgq.lib.sgqd_rope_kv_store_int8(qkv, stride, t, heads, cos, sin, rows, pos, ps, n_new, offset, q, qs, c, None)


def test_store_arguments(sgq):
    assert store(sgq, None) == 1
    assert store(sgq, cache(sgq, batch=-1)) == 2 and store(sgq, cache(sgq, kv=0)) == 2 and store(sgq, cache(sgq, max_seq=0)) == 2
    assert store(sgq, cache(sgq, max_seq=2 ** 31)) == 2 and store(sgq, cache(sgq, batch=2 ** 40)) == 2
    assert store(sgq, cache(sgq, dim=12)) == 2 and store(sgq, cache(sgq, dim=264)) == 2 and store(sgq, cache(sgq, dim=0)) == 2
    assert store(sgq, cache(sgq), heads=3) == 2 and store(sgq, cache(sgq), heads=0) == 2 and store(sgq, cache(sgq), heads=2 ** 20) == 2
    assert store(sgq, cache(sgq), t=-1) == 2 and store(sgq, cache(sgq), t=2 ** 31) == 2 and store(sgq, cache(sgq), t=2 ** 30) == 2
    assert store(sgq, cache(sgq), stride=1020) == 2 and store(sgq, cache(sgq), qs=508) == 2
    assert store(sgq, cache(sgq), ps=2) == 3 and store(sgq, cache(sgq), rows=15) == 2
    assert store(sgq, cache(sgq), q=ONE) == 3                                        # in place with another stride
    for missing in ("qkv", "cos", "sin", "pos", "q"):
        assert store(sgq, cache(sgq), **{missing: None}) == 1, missing
    for missing in ("k", "ks", "v", "vs"):
        assert store(sgq, cache(sgq, **{missing: None})) == 1, missing
    assert store(sgq, cache(sgq, k=260)) == 6 and store(sgq, cache(sgq, vs=257)) == 6
    for off in ("qkv", "cos", "sin", "q"):
        assert store(sgq, cache(sgq), **{off: ODD}) == 6, off
    assert store(sgq, cache(sgq), stride=1026) == 6 and store(sgq, cache(sgq), qs=514) == 6
    assert store(sgq, cache(sgq, batch=0, k=None)) == 0 and store(sgq, cache(sgq), t=0, qkv=None) == 0


def load(sgq, c, rows=16, batch=2, k=ONE, v=TWO, out_rows=16, row0=0):
    return sgq.lib.sgqd_kv_load_int8(c, rows, batch, k, v, out_rows, row0, None)


def test_load_arguments(sgq):
    assert load(sgq, None) == 1 and load(sgq, cache(sgq, dim=20)) == 2
    assert load(sgq, cache(sgq), rows=17) == 2 and load(sgq, cache(sgq), rows=-1) == 2
    assert load(sgq, cache(sgq), batch=3) == 2 and load(sgq, cache(sgq), batch=-1) == 2
    assert load(sgq, cache(sgq), row0=-1) == 2 and load(sgq, cache(sgq), row0=1) == 2 and load(sgq, cache(sgq), row0=2 ** 62) == 2
    assert load(sgq, cache(sgq), k=None) == 1 and load(sgq, cache(sgq), v=None) == 1 and load(sgq, cache(sgq, ks=None)) == 1
    assert load(sgq, cache(sgq), k=ODD) == 6
    assert load(sgq, cache(sgq), rows=0, k=None) == 0 and load(sgq, cache(sgq, batch=1), batch=0, k=None) == 0
    big = cache(sgq, batch=1, kv=65535, max_seq=2 ** 31 - 1, dim=256)
    assert load(sgq, big, rows=2 ** 31 - 1, batch=1000, out_rows=2 ** 31 - 1) == 2     # more blocks than a launch takes


def decode(sgq, c, prefix=False, p=None, qkv=ONE, stride=1024, heads=4, cos=ONE, sin=ONE, rows=16, pos=ONE, ps=1, length=ONE, out=TWO, os=512,
           planes=None, nb=0, ws=ONE, wb=1 << 30):
    if prefix:
        return sgq.lib.sgqd_attn_decode_prefix_int8(qkv, stride, heads, cos, sin, rows, pos, ps, c, p, length, out, os, planes, nb, ws, wb, None)
    return sgq.lib.sgqd_attn_decode_int8(qkv, stride, heads, cos, sin, rows, pos, ps, c, out, os, planes, nb, ws, wb, None)


@pytest.mark.parametrize("prefix", [False, True])
def test_decode_arguments(sgq, prefix):
    def call(c=cache(sgq), **kw):
        return decode(sgq, c, prefix, cache(sgq, batch=1, max_seq=32) if prefix else None, **{"rows": 48 if prefix else 16, **kw})
    assert call(c=None) == 1 and call(c=cache(sgq, dim=96)) == 4 and call(c=cache(sgq, dim=256)) == 4 and call(c=cache(sgq, kv=-2)) == 2
    assert call(heads=5) == 2 and call(heads=-4) == 2 and call(stride=1000) == 2 and call(os=500) == 2 and call(ps=-1) == 3
    assert call(rows=47 if prefix else 15) == 2
    for missing in ("qkv", "cos", "sin", "pos", "out"):
        assert call(**{missing: None}) == 1, missing
    assert call(c=cache(sgq, vs=None)) == 1 and call(c=cache(sgq, v=264)) == 6 and call(qkv=ODD) == 6 and call(stride=1025) == 6 and call(sin=ODD) == 6
    assert call(planes=ONE, nb=16) == 5 and call(c=cache(sgq, batch=17), planes=ONE, nb=1 << 20) == 4
    assert call(c=cache(sgq, batch=0, k=None), out=None) == 0


@pytest.mark.parametrize("at,stride,overlaps", [
    (1020, 1600, True), (-508, 1600, True), (1600, 1600, True), (1500, 1600, True),          # the same rows' columns, the next row's, over a row's end
    (1024, 1600, False), (1088, 1600, False), (2624, 1600, False), (-512, 1600, False),      # behind the columns, or in front
    (1024, 1604, True), (2624, 1604, False), (-512 - 1604, 1604, False)])                    # spaced otherwise
def test_outputs_that_overlap_the_rows_they_are_made_of(sgq, at, stride, overlaps):
    """Two rows of 1024 floats, 1600 apart, outputs `at` floats behind.  What does not overlap comes as far as the next check."""
    qkv, out = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 4 * at)
    if overlaps:                       # (nothing would refuse the others, on a GPU)
        assert store(sgq, cache(sgq), qkv=qkv, stride=1600, q=out, qs=stride) == 3
    assert decode(sgq, cache(sgq), qkv=qkv, stride=1600, out=out, os=stride, planes=ONE, nb=16) == (3 if overlaps else 5)


def test_prefix_arguments(sgq):
    c = cache(sgq)
    assert decode(sgq, c, True, None, rows=48) == 1
    for p in (cache(sgq, batch=2), cache(sgq, batch=1, kv=4), cache(sgq, batch=1, dim=64), cache(sgq, batch=0)):
        assert decode(sgq, c, True, p, rows=48) == 2
    good = cache(sgq, batch=1, max_seq=32)
    assert decode(sgq, c, True, good, rows=48, length=None) == 1
    assert decode(sgq, c, True, cache(sgq, batch=1, max_seq=32, k=None), rows=48) == 1
    need = sgq.lib.sgqd_attn_decode_prefix_int8_workspace_bytes(2, 4, 2, 128, 16, 32)
    assert need > 0
    assert decode(sgq, c, True, good, rows=48, ws=None) == 5 and decode(sgq, c, True, good, rows=48, wb=need - 1) == 5
    assert decode(sgq, c, True, good, rows=48, ws=C.c_void_p(272)) == 5


def test_workspace_queries(sgq):
    own, prefix = sgq.lib.sgqd_attn_decode_int8_workspace_bytes, sgq.lib.sgqd_attn_decode_prefix_int8_workspace_bytes
    for bad in ((0, 4, 2, 128, 32), (2, 4, 3, 128, 32), (2, 4, 0, 128, 32), (2, 4, 2, 96, 32), (2, 4, 2, 128, 0), (-1, 4, 2, 128, 32), (2, -4, 2, 128, 32),
                (2, 2 ** 20, 2, 128, 32), (2, 4, 2, 128, 2 ** 30 + 1), (2 ** 31, 4, 2, 128, 32)):
        assert own(*bad) == 0 and prefix(*bad, 64) == 0, bad
    assert prefix(2, 4, 2, 128, 32, 0) == 0 and prefix(2, 4, 2, 128, 32, -1) == 0 and prefix(2, 4, 2, 128, 32, 2 ** 30 + 1) == 0
    assert own(1, 16, 16, 128, 640) == 0                                   # a short cache: joined inside a cluster of CTAs
    assert own(32, 32, 8, 128, 8192) == 0                                  # and so are those of many sequences
    need = own(2, 32, 8, 128, 65536)                                       # few long ones: partial results in the workspace
    assert need > 0 and prefix(2, 32, 8, 128, 65536, 1024) > need
    long = cache(sgq, batch=2, kv=8, max_seq=65536)
    args = dict(stride=6144, heads=32, os=4096, rows=65536)
    assert decode(sgq, long, ws=None, **args) == 5 and decode(sgq, long, wb=need - 1, **args) == 5 and decode(sgq, long, ws=C.c_void_p(264), **args) == 5
    assert decode(sgq, cache(sgq, max_seq=2 ** 30 + 1), rows=2 ** 31) == 2


# ---- the Python calls -----------------------------------------------------------------------------------------------
B, HEADS, KV, DIM, S = 2, 4, 2, 64, 16
WIDTH = (HEADS + 2 * KV) * DIM


def given(sgq, **kw):
    g = {"qkv": torch.zeros(B, 1, WIDTH), "cache": sgq.KVCacheInt8.empty(B, KV, S, DIM, "cpu"), "cos": torch.zeros(S, DIM // 2), "sin": torch.zeros(S, DIM // 2),
         "pos": torch.zeros(B, dtype=torch.int32), "n_heads": HEADS}
    g.update(kw)
    return g


SHARED = [dict(qkv=torch.zeros(B, 1, WIDTH - 1)), dict(qkv=torch.zeros(B + 1, 1, WIDTH)), dict(qkv=torch.zeros(WIDTH)), dict(n_heads=3), dict(n_heads=0),
          dict(cos=torch.zeros(S, DIM)), dict(sin=torch.zeros(S + 1, DIM // 2)), dict(cos=torch.zeros(S, DIM // 2).double(), sin=torch.zeros(S, DIM // 2)),
          dict(pos=torch.zeros(3, dtype=torch.int32)), dict(pos=torch.zeros(2, dtype=torch.int64)), dict(pos=torch.zeros(1, 2, dtype=torch.int32)),
          dict(pos=torch.zeros(4, dtype=torch.int32)[::2]), dict(pos=torch.zeros(0, dtype=torch.int32))]


@pytest.mark.parametrize("wrong", range(len(SHARED)))
@pytest.mark.parametrize("name", ["rope_kv_store_int8", "attn_decode_int8", "attn_decode_prefix_int8"])
def test_shapes_are_refused_without_a_device(sgq, name, wrong):
    kw = given(sgq, **SHARED[wrong])
    if name == "attn_decode_prefix_int8":
        kw.update(prefix=sgq.KVCacheInt8.empty(1, KV, 8, DIM, "cpu"), prefix_len=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        getattr(sgq, name)(**kw)


def test_host_tensors_are_refused(sgq):
    with pytest.raises(ValueError):
        sgq.rope_kv_store_int8(**given(sgq))
    with pytest.raises(ValueError):
        sgq.attn_decode_int8(**given(sgq))
    with pytest.raises(ValueError):
        sgq.kv_load_int8(given(sgq)["cache"], 4)
    with pytest.raises(ValueError):
        sgq.attn_decode_prefix_int8(**given(sgq), prefix=sgq.KVCacheInt8.empty(1, KV, 8, DIM, "cpu"), prefix_len=torch.zeros(1, dtype=torch.int32))


def test_broken_caches_are_refused(sgq):
    good = sgq.KVCacheInt8.empty(B, KV, S, DIM, "cpu")
    for field, value in [("k_codes", good.k_codes.float()), ("v_codes", good.v_codes[:, :, :-1]), ("k_scales", good.k_scales[:, :1]),
                         ("v_scales", good.v_scales.double()), ("v_scales", good.v_scales.unsqueeze(-1)), ("k_codes", good.k_codes[0]),
                         ("v_codes", good.v_codes.transpose(1, 2).contiguous().transpose(1, 2)),
                         ("k_scales", good.k_scales.transpose(0, 1).contiguous().transpose(0, 1))]:
        broken = sgq.KVCacheInt8(good.k_codes, good.k_scales, good.v_codes, good.v_scales)
        setattr(broken, field, value)
        with pytest.raises(RuntimeError):
            sgq.attn_decode_int8(**given(sgq, cache=broken))
        with pytest.raises(RuntimeError):
            sgq.kv_load_int8(broken, 1)
    broken = sgq.KVCacheInt8(good.k_codes, None, good.v_codes, good.v_scales)
    with pytest.raises(TypeError):
        sgq.kv_load_int8(broken, 1)
    with pytest.raises(AttributeError):
        sgq.kv_load_int8(object(), 1)


def test_optional_arguments_are_refused(sgq):
    for kw in (dict(n_new=torch.zeros(3, dtype=torch.int32)), dict(n_new=torch.zeros(2)), dict(rope_offset=torch.zeros(2, dtype=torch.int32)),
               dict(rope_offset=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            sgq.rope_kv_store_int8(**given(sgq), **kw)
    c = given(sgq)["cache"]
    for kw in (dict(rows=S + 1), dict(rows=-1), dict(rows=4, batch=3), dict(rows=4, row0=1), dict(rows=4, k_out=torch.zeros(B, KV, 4, DIM)),
               dict(rows=4, k_out=torch.zeros(B, KV, 4, DIM), v_out=torch.zeros(B, KV, 5, DIM)),
               dict(rows=4, k_out=torch.zeros(B, KV, 4, DIM), v_out=torch.zeros(B, KV, 4, DIM), row0=1),
               dict(rows=4, k_out=torch.zeros(B, KV, 4, DIM).double(), v_out=torch.zeros(B, KV, 4, DIM).double())):
        with pytest.raises(RuntimeError):
            sgq.kv_load_int8(c, **kw)
    first = sgq.KVCacheInt8.empty(1, KV, 8, DIM, "cpu")
    for kw in (dict(prefix=sgq.KVCacheInt8.empty(2, KV, 8, DIM, "cpu"), prefix_len=torch.zeros(1, dtype=torch.int32)),
               dict(prefix=sgq.KVCacheInt8.empty(1, KV + 1, 8, DIM, "cpu"), prefix_len=torch.zeros(1, dtype=torch.int32)),
               dict(prefix=first, prefix_len=torch.zeros(2, dtype=torch.int32)), dict(prefix=first, prefix_len=torch.zeros(1))):
        with pytest.raises(RuntimeError):
            sgq.attn_decode_prefix_int8(**given(sgq), **kw)
    with pytest.raises(TypeError):
        sgq.attn_decode_prefix_int8(**given(sgq), prefix=first, prefix_len=3)
    with pytest.raises(RuntimeError):
        sgq.attn_decode_int8(**given(sgq, qkv=torch.zeros(B, 2, WIDTH)))


@pytest.mark.parametrize("kw", [dict(kv_cache="int4"), dict(kv_cache="int8", world=2), dict(kv_cache="int8", heads=8), dict(max_prefix=4),
                                dict(kv_cache="int8", max_prefix=-1)])
def test_the_decoder_refuses_caches_it_cannot_serve(sgq, kw):
    import importlib
    nl = importlib.import_module("sgq_b200.nanollama")
    cfg = nl.NanoLlamaConfig(dim=256, n_layers=1, n_heads=kw.pop("heads", 2), hidden=512, vocab=512, max_seq=16)
    with pytest.raises(ValueError):
        nl.NanoLlamaInt4(cfg, "cpu", 1, **kw)
