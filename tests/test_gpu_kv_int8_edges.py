"""The INT8 key/value cache at the edges of what its calls take: parts of a kernel that have nothing to do, inputs near the ends of the
fp32 range, rows that must not be missed."""
import ctypes as C

import numpy as np
import pytest
import torch

import kv_int8_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sgq():
    from __graft_entry__ import load_package
    return load_package()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def to_gpu(sgq, c):
    return sgq.KVCacheInt8(**{k: dev(v) for k, v in c.items()})


def cache_of(keys, values):
    c = {}
    for name, rows in (("k", keys), ("v", values)):
        c[name + "_codes"], c[name + "_scales"] = plain.held(np.asarray(rows, np.float32))
    return c


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prefix_len", [0, 1, 128, 129, 700])
def test_prefixes_far_below_their_capacity(sgq, prefix_len, dim):
    """40 and 130 query rows per kv head and room for 4000 tokens: most parts of the prefix kernel have no tile.  They still ask for
    their queries' rows, have to wait for them before they read them, and may not end before they have arrived."""
    r = np.random.default_rng(prefix_len + dim)
    for B, heads, kv in ((20, 4, 2), (65, 2, 1)):
        S, room = 24, 4000
        rows = lambda n, b: r.standard_normal((b, kv, n, dim))  # noqa: E731
        own, first = cache_of(rows(S, B), rows(S, B)), cache_of(rows(room, 1), rows(room, 1))
        qkv = r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32)
        cos, sin = plain.tables(S + room, dim)
        pos = [(7 * b) % (S + 2) - 1 for b in range(B)]
        want, _, tol = plain.decode(qkv, own, cos, sin, pos, heads, first, prefix_len)
        args = (to_gpu(sgq, first), ints(prefix_len), dev(cos), dev(sin), ints(*pos), heads)
        got = [sgq.attn_decode_prefix_int8(dev(qkv), to_gpu(sgq, own), *args) for _ in range(3)]
        assert all(torch.equal(g, got[0]) for g in got)
        off = np.abs(got[0].cpu().numpy() - want)
        assert (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()
    assert sgq.device_status() == 0


def test_tensors_side_by_side_in_one_buffer(sgq):
    """Everything a step needs next to one another without a gap; keys and values read back into alternate halves of one tensor."""
    B, heads, kv, dim, S = 2, 4, 2, 64, 16
    r = np.random.default_rng(5)
    host = cache_of(r.standard_normal((B, kv, S, dim)), r.standard_normal((B, kv, S, dim)))
    qkv = r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32)
    cos, sin = (dev(t) for t in plain.tables(S, dim))
    want = sgq.attn_decode_int8(dev(qkv), to_gpu(sgq, host), cos, sin, ints(9, 15), heads)
    codes, scales, out = B * kv * S * dim, B * kv * S, B * heads * dim
    buf = torch.zeros(2 * codes + 8 * scales + 4 * (qkv.size + out), dtype=torch.uint8, device="cuda")
    part, at = [], 0
    for n, dtype, shape in ((codes, torch.int8, (B, kv, S, dim)), (4 * scales, torch.float32, (B, kv, S)), (codes, torch.int8, (B, kv, S, dim)),
                            (4 * scales, torch.float32, (B, kv, S)), (4 * qkv.size, torch.float32, qkv.shape), (4 * out, torch.float32, (B, heads * dim))):
        part.append(buf[at:at + n].view(dtype).view(shape))
        at += n
    cache = sgq.KVCacheInt8(*part[:4])
    for name in host:
        getattr(cache, name).copy_(dev(host[name]))
    part[4].copy_(dev(qkv))
    assert torch.equal(sgq.attn_decode_int8(part[4], cache, cos, sin, ints(9, 15), heads, out=part[5]), want)
    k, v = sgq.kv_load_int8(cache, S)
    both = torch.zeros(B, kv, 2 * S, dim, device="cuda")
    c = sgq.CacheInt8(*(getattr(cache, n).data_ptr() for n in ("k_codes", "k_scales", "v_codes", "v_scales")), B, kv, S, dim)
    sgq.check(sgq.lib.sgqd_kv_load_int8(C.byref(c), S, B, C.c_void_p(both.data_ptr()), C.c_void_p(both.data_ptr() + S * dim * 4), 2 * S, 0,
                                        C.c_void_p(torch.cuda.current_stream().cuda_stream)), "sgqd_kv_load_int8")
    assert torch.equal(both[:, :, :S], k) and torch.equal(both[:, :, S:], v)
    with pytest.raises(sgq.SgqError):
        sgq.kv_load_int8(cache, S, k_out=k, v_out=k)
    one = sgq.KVCacheInt8(*(t[:1].clone() for t in part[:4]))
    long = [dev(t) for t in plain.tables(2 * S, dim)]
    with pytest.raises(sgq.SgqError):
        sgq.attn_decode_prefix_int8(part[4][:1], one, one, ints(4), *long, ints(4), heads)
