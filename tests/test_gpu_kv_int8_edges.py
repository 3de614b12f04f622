"""The INT8 key/value cache at the edges of what its calls take: parts of a kernel that have nothing to do, inputs near the ends of the
fp32 range, rows that must not be missed."""
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
