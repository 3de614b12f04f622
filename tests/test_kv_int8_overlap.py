"""Calls of the INT8 key/value cache whose tensors share memory that one of them writes, or that lie off the grid of their type: refused
before a device is touched.  Every call here is one; any other would be launched on these made-up addresses."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def sgq():
    from __graft_entry__ import load_package
    return load_package()


B, HEADS, KV, DIM, S, P = 2, 4, 2, 128, 16, 32
CODES, SCALES = B * KV * S * DIM, B * KV * S * 4
AT = {name: (i + 1) << 24 for i, name in enumerate(("k", "ks", "v", "vs", "pk", "pks", "pv", "pvs", "qkv", "out", "planes", "ws", "tables", "v_out"))}
BAD_ARGUMENT, ALIGNMENT = 3, 6


def ptr(x):
    return C.c_void_p(x)


def own(sgq, a):
    return C.byref(sgq.CacheInt8(a["k"], a["ks"], a["v"], a["vs"], B, KV, S, DIM))


def first(sgq, a):
    return C.byref(sgq.CacheInt8(a["pk"], a["pks"], a["pv"], a["pvs"], 1, KV, P, DIM))


def store(sgq, a):
    return sgq.lib.sgqd_rope_kv_store_int8(ptr(a["qkv"]), 1024, 1, HEADS, ptr(a["tables"]), ptr(a["tables"]), S, ptr(a["tables"]), 1, None, None,
                                           ptr(a["out"]), 512, own(sgq, a), None)


def decode(sgq, a, prefix):
    planes = sgq.prepared_x_bytes(B, HEADS * DIM)
    if not prefix:
        return sgq.lib.sgqd_attn_decode_int8(ptr(a["qkv"]), 1024, HEADS, ptr(a["tables"]), ptr(a["tables"]), S, ptr(a["tables"]), 1, own(sgq, a),
                                             ptr(a["out"]), 512, ptr(a["planes"]), planes, None, 0, None)
    return sgq.lib.sgqd_attn_decode_prefix_int8(ptr(a["qkv"]), 1024, HEADS, ptr(a["tables"]), ptr(a["tables"]), S + P, ptr(a["tables"]), 1, own(sgq, a),
                                                first(sgq, a), ptr(a["tables"]), ptr(a["out"]), 512, ptr(a["planes"]), planes, ptr(a["ws"]), 1 << 20, None)


# (what is moved, onto the last 256 bytes of what or a few more, its size)
ROWS = B * 1024 * 4
OWN = [("k", "v", CODES), ("ks", "k", CODES), ("vs", "ks", SCALES), ("v", "vs", SCALES)]
BOTH = [("out", "k", CODES), ("out", "vs", SCALES), ("qkv", "v", CODES), ("ks", "qkv", ROWS)]
PLANES = [("planes", "out", B * 512 * 4), ("planes", "qkv", ROWS), ("planes", "ks", SCALES)]
PREFIX = [("pk", "k", CODES), ("pvs", "vs", SCALES), ("pv", "k", CODES), ("k", "pks", KV * P * 4), ("out", "pk", KV * P * DIM), ("ws", "pv", KV * P * DIM),
          ("ws", "out", B * 512 * 4), ("ws", "qkv", ROWS), ("ws", "v", CODES), ("planes", "pvs", KV * P * 4)]


def moved(what, onto, size):
    return {**AT, what: AT[onto] + size - 16 - (size - 16) % 256}          # keeps every alignment


@pytest.mark.parametrize("what,onto,size", OWN + BOTH)
def test_store(sgq, what, onto, size):
    assert store(sgq, moved(what, onto, size)) == BAD_ARGUMENT


@pytest.mark.parametrize("what,onto,size", OWN + BOTH + PLANES)
def test_decode(sgq, what, onto, size):
    assert decode(sgq, moved(what, onto, size), False) == BAD_ARGUMENT


@pytest.mark.parametrize("what,onto,size", OWN + BOTH + PLANES + PREFIX)
def test_decode_behind_a_prefix(sgq, what, onto, size):
    assert decode(sgq, moved(what, onto, size), True) == BAD_ARGUMENT


def test_one_cache_as_both(sgq):
    """A cache of one sequence is a prefix by its shape; the call would append to what it reads."""
    c = C.byref(sgq.CacheInt8(AT["k"], AT["ks"], AT["v"], AT["vs"], 1, KV, S, DIM))
    assert sgq.lib.sgqd_attn_decode_prefix_int8(ptr(AT["qkv"]), 1024, HEADS, ptr(AT["tables"]), ptr(AT["tables"]), 2 * S, ptr(AT["tables"]), 1, c, c,
                                                ptr(AT["tables"]), ptr(AT["out"]), 512, None, 0, ptr(AT["ws"]), 1 << 20, None) == BAD_ARGUMENT


@pytest.mark.parametrize("k,v,rows,room,row0", [
    (0, 0, S, S, 0), (0, 0, 1, S, 5), (0, 3 * DIM * 4, 4, S, 0), (3 * DIM * 4, 0, 4, S, 2),          # the same tensor, rows that meet
    (0, (B * KV * S - 1) * DIM * 4, S, S, 0), (0, (S - 1) * DIM * 4, 2, S, 0)])                       # its last row, the next head's first
def test_load_into_one_tensor_twice(sgq, k, v, rows, room, row0):
    assert sgq.lib.sgqd_kv_load_int8(own(sgq, AT), rows, B, ptr(AT["out"] + k), ptr(AT["out"] + v), room, row0, None) == BAD_ARGUMENT


@pytest.mark.parametrize("name,size", [("k", CODES), ("ks", SCALES), ("v", CODES), ("vs", SCALES)])
def test_load_over_the_cache(sgq, name, size):
    assert sgq.lib.sgqd_kv_load_int8(own(sgq, AT), S, B, ptr(AT[name] + size - 64), ptr(AT["v_out"]), S, 0, None) == BAD_ARGUMENT
    assert sgq.lib.sgqd_kv_load_int8(own(sgq, AT), S, B, ptr(AT["v_out"]), ptr(AT[name]), S, 0, None) == BAD_ARGUMENT


@pytest.mark.parametrize("off", [1, 2, 3])
def test_small_vectors_off_their_grid(sgq, off):
    p, t, q = ptr(AT["tables"] + off), ptr(AT["tables"]), ptr(AT["qkv"])
    for pos, n_new, offset in ((p, None, None), (t, p, None), (t, None, p)):
        assert sgq.lib.sgqd_rope_kv_store_int8(q, 1024, 1, HEADS, t, t, S, pos, 1, n_new, offset, ptr(AT["out"]), 512, own(sgq, AT), None) == ALIGNMENT
    for pos, out in ((p, ptr(AT["out"])), (t, ptr(AT["out"] + off))):
        assert sgq.lib.sgqd_attn_decode_int8(q, 1024, HEADS, t, t, S, pos, 1, own(sgq, AT), out, 512, None, 0, None, 0, None) == ALIGNMENT
    assert sgq.lib.sgqd_attn_decode_prefix_int8(q, 1024, HEADS, t, t, S + P, t, 1, own(sgq, AT), first(sgq, AT), p, ptr(AT["out"]), 512, None, 0,
                                                ptr(AT["ws"]), 1 << 20, None) == ALIGNMENT
