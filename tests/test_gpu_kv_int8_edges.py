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


# ---- near the ends of the fp32 range --------------------------------------------------------------------------------------
# sequences, heads, kv heads, capacity and position, length of the shared prefix: a cluster of CTAs per head (4 and 8 queries), a cache dealt
# out to all warps, and behind a prefix 4, 16, 32 and 40 query rows per kv head (8 rows per warp, one to four warps side by side; tcgen05)
FORMS = [(2, 4, 2, 130, 99, 0), (1, 8, 1, 300, 299, 0), (1, 4, 1, 20000, 700, 0), (2, 4, 2, 40, 9, 200), (4, 8, 2, 40, 9, 200), (8, 8, 2, 40, 9, 200), (10, 8, 2, 40, 9, 200)]


class Step:
    """A decode step on N(0, 1) rows times q_size, k_size and v_size (the cache's, the prefix's and the new token's alike)."""

    def __init__(self, form, dim, q_size, k_size, v_size, seed=0, shape_v=lambda v: v):
        self.B, self.heads, self.kv, self.S, self.pos, self.P = form
        self.dim = dim
        r = np.random.default_rng(seed + dim + self.S + self.P + self.B)
        f = lambda *shape: r.standard_normal(shape)  # noqa: E731
        self.qkv = f(self.B, self.heads + 2 * self.kv, dim)
        for at, size in ((slice(0, self.heads), q_size), (slice(self.heads, self.heads + self.kv), k_size), (slice(self.heads + self.kv, None), v_size)):
            self.qkv[:, at] *= size
        self.qkv[:, self.heads + self.kv:] = shape_v(self.qkv[:, self.heads + self.kv:])
        self.qkv = self.qkv.astype(np.float32)
        self.cos, self.sin = plain.tables(self.S + self.P, dim)
        keys, first = f(self.B, self.kv, self.S, dim) * k_size, f(1, self.kv, self.P, dim) * k_size
        at = self.P + self.pos
        like = plain.turned(self.qkv[:, :self.heads:self.heads // self.kv].astype(np.float64), self.cos[at], self.sin[at]) * (k_size / q_size)
        keys[:, :, [1, self.pos - 1]] = like[:, :, None]         # keys along the first query of each kv head (of sequence 0 in the prefix), twice
        if self.P:
            first[0][:, [2, self.P - 1]] = like[0][:, None]
        self.own = cache_of(keys, shape_v(f(self.B, self.kv, self.S, dim) * v_size))
        self.first = cache_of(first, shape_v(f(1, self.kv, self.P, dim) * v_size)) if self.P else None

    def want(self):
        return plain.decode(self.qkv.reshape(self.B, -1), self.own, self.cos, self.sin, [self.pos], self.heads, self.first, self.P)

    def run(self, sgq):
        x, cache, rest = dev(self.qkv.reshape(self.B, -1)), to_gpu(sgq, self.own), (dev(self.cos), dev(self.sin), ints(self.pos), self.heads)
        if self.first is None:
            return sgq.attn_decode_int8(x, cache, *rest).cpu().numpy()
        return sgq.attn_decode_prefix_int8(x, cache, to_gpu(sgq, self.first), ints(self.P), *rest).cpu().numpy()

    def check(self, sgq):
        want, _, tol = self.want()
        got = self.run(sgq)
        assert np.isfinite(want).all() and np.isfinite(tol).all()
        off = np.abs(got - want) / tol
        assert np.isfinite(got).all() and off.max() <= 1, off.max()

    def rows(self, b, h):
        """The positions that query head h of sequence b attends to: keys and values in 64 bits, and its rotated query."""
        hk, at = h // (self.heads // self.kv), self.P + self.pos
        out = []
        for name, new in (("k", plain.turned(self.qkv[b, self.heads + hk], self.cos[at], self.sin[at])), ("v", self.qkv[b, self.heads + self.kv + hk])):
            parts = [self.first[name + "_codes"][0, hk].astype(np.float64) * self.first[name + "_scales"][0, hk, :, None]] if self.P else []
            parts.append(self.own[name + "_codes"][b, hk, :self.pos].astype(np.float64) * self.own[name + "_scales"][b, hk, :self.pos, None])
            codes, scale = plain.held(new)
            parts.append(codes[None].astype(np.float64) * np.float64(scale))
            out.append(np.concatenate(parts))
        q = plain.turned(self.qkv[b, h].astype(np.float64), self.cos[at].astype(np.float64), self.sin[at].astype(np.float64))
        return out[0], out[1], q


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("q_size,k_size", [(1.0, 1.0), (1.2e-30, 4e30), (1e-25, 1e25), (1e-31, 1e31), (2e-34, 1e34), (1e-36, 1e36)])
def test_large_keys_and_small_queries(sgq, form, dim, q_size, k_size):
    """Scores of ordinary size whose factors are far from one: the bound of tests/kv_int8_plain.py, which is relative to both."""
    Step(form, dim, q_size, k_size, 1.0).check(sgq)


def winners(sgq, step):
    """Where a query's largest scores are far ahead, their positions take all the weight and, having the same key, share it alike: out is
    the mean of their values, within the weights' fixed point, their exponential, the joining of up to six and the division:
    16 * 2^-24 of the largest.  Heads whose lead is not beyond any rounding are passed over."""
    got = step.run(sgq).reshape(step.B, step.heads, step.dim)
    seen = shared = 0
    for b in range(step.B):
        for h in range(step.heads):
            k, v, q = step.rows(b, h)
            s = k @ q / np.sqrt(step.dim)
            lead = (k == k[np.argmax(s)]).all(-1)
            room = 16 * 2.0 ** -24 * np.abs(q).max() * np.abs(k).sum(-1).max() / np.sqrt(step.dim)
            if s.max() - s[~lead].max() > room + 100:
                assert np.abs(got[b, h] - v[lead].mean(0)).max() <= 16 * 2.0 ** -24 * np.abs(v[lead]).max(), (b, h)
                seen, shared = seen + 1, shared + (lead.sum() > 1)
    assert seen > step.B * step.heads / 2 and shared >= step.kv, "choose other inputs"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("q_size,k_size", [(1e4, 1.0), (1e15, 1e-7), (1.0, 1e12), (3e30, 1.0), (1e30, 1e-3), (1.2e36, 1e-6)])
def test_scores_that_leave_the_largest_alone(sgq, form, dim, q_size, k_size):
    """Among them large queries times small keys, whose scores of 1e30 are fp32 numbers."""
    winners(sgq, Step(form, dim, q_size, k_size, 1.0))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS[3:])
@pytest.mark.parametrize("size", [20.0, 60.0, 200.0, 2000.0])
def test_steep_scores_behind_a_prefix(sgq, form, dim, size):
    """Largest scores of 300 to 20000: within the bound of an fp32 evaluation on both sides of the size from which the tcgen05 kernel rounds
    them one by one."""
    Step(form, dim, size, 1.0, 1.0).check(sgq)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS + [(1, 4, 1, 20000, 19999, 0), (2, 8, 4, 900, 899, 0), (33, 1, 1, 40, 9, 3000), (3, 1, 1, 40, 9, 3000)])
@pytest.mark.parametrize("q_size", [1e-3, 1.5])
@pytest.mark.parametrize("v_size", [1e-7, 1.0, 1e38])
@pytest.mark.parametrize("positive", [False, True])
def test_values_of_any_size(sgq, form, dim, q_size, v_size, positive):
    """Up to 3e38: many of one sign, whose sum is no fp32 number, or a single one whose weight and scale are large together."""
    shape = lambda v: np.clip(np.abs(v) if positive else v, -3e38, 3e38)  # noqa: E731
    Step(form, dim, q_size, 1.0, v_size, shape_v=shape).check(sgq)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_scores_beyond_the_fp32_range(sgq, form, dim):
    """Query heads 0 and 1 of the last sequence meet keys that make every score overflow, below and above; NaN, not a number that looks
    like an output.  So does a query value beyond 2^122 (head 2).  The others are as ever."""
    step = Step(form, dim, 1.0, 1.0, 1.0)
    b, size = step.B - 1, np.float32(1e5)
    along = np.ones(dim, np.float32)
    at = step.P + step.pos
    turn = lambda x: plain.turned(x, step.cos[at], -step.sin[at])  # noqa: E731  (rotates back)
    for cache, i in ((step.own, b), (step.first, 0)):
        if cache is not None:                                   # keys with a large common part: q . k is that of the part
            keys = cache["k_codes"][i].astype(np.float32) * cache["k_scales"][i][..., None] + size
            cache["k_codes"][i], cache["k_scales"][i] = plain.held(keys)
    step.qkv[b, step.heads:step.heads + step.kv] = turn(along * size)
    step.qkv[b, 0], step.qkv[b, 1] = turn(along * np.float32(-1e36)), turn(along * np.float32(1e36))
    step.qkv[b, 2] = turn(along * np.float32(1e37))
    want, _, tol = step.want()
    got = step.run(sgq).reshape(step.B, step.heads, dim)
    assert np.isnan(got[b, :3]).all()
    fine = np.ones(got.shape, bool)
    fine[b, :3] = False
    off = np.abs(got - want.reshape(got.shape))
    assert (off <= tol.reshape(got.shape))[fine].all()


# ---- every row, once ------------------------------------------------------------------------------------------------------
# sequences, heads, kv heads, capacity, positions, length and capacity of the prefix
ROWS = [(8, 16, 16, 640, [575], 0, 0), (1, 16, 16, 9000, [8999], 0, 0), (2, 16, 2, 9000, [8999, 4500], 0, 0), (40, 32, 32, 600, [599], 0, 0),
        (33, 8, 8, 1500, [1499], 0, 0), (1, 4, 1, 40000, [39999], 0, 0), (5, 10, 2, 700, [699, 64, -1, 127, 0], 0, 0),
        (1, 4, 2, 80000, [70001], 0, 0), (4, 32, 8, 4096, [4095, 1, 63, 2049], 0, 0), (2, 32, 4, 30000, [29999, 127], 0, 0),
        (6, 6, 6, 7000, [6999, -1, 64, 128, -1, 3500], 0, 0), (30, 4, 1, 3000, [100 * i - 1 for i in range(30)], 0, 0),
        (2, 4, 2, 40, [33, 2], 20011, 20480), (4, 12, 4, 40, [33, 0, 39, -1], 4999, 5000), (7, 4, 1, 40, [33], 9001, 9100),
        (12, 4, 1, 40, [33], 20011, 20480), (50, 4, 1, 40, [20], 5000, 5000), (35, 16, 8, 300, [299], 1025, 4000), (10, 40, 10, 12, [11], 129, 129),
        (16, 16, 16, 64, [63], 777, 800), (3, 6, 6, 7000, [6999, 5, 100], 700, 720)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("B,heads,kv,S,pos,P,room", ROWS)
def test_every_row_counts_once(sgq, B, heads, kv, S, pos, P, room, dim):
    """Keys of zero: all n positions weigh 1 / n.  Row t holds one value, 127 s_t in column t mod dim with s_t between 0.5 and 1, so a row that is
    missed, or read twice, changes its column by s_t of the sum of about n / dim such, relative to what stands there.

    All terms are positive, so errors are relative too: 24 * 2^-24 for a term (the weight's fixed point, half a step of 1 / 4194000 of the
    largest, which is at most twice the term: 4; its exponential and the division for its unit, 2 ulp each: 8; products, conversions
    and the final division: the rest), and 2^-24 for each addition in a row, of outputs and of weights.  A warp takes every fourth step of at
    least 32 positions or less (128 positions a step in the tcgen05 kernel), so that n / 128 + 1 additions follow one another, and 40 join parts."""
    r = np.random.default_rng(S + P + B + dim)

    def rows(batch, n, first):
        codes, scales = np.zeros((batch, kv, n, dim), np.int8), r.uniform(0.5, 1.0, (batch, kv, n)).astype(np.float32)
        codes[:, :, np.arange(n), (first + np.arange(n)) % dim] = 127
        return {"k_codes": np.zeros_like(codes), "k_scales": np.ones_like(scales), "v_codes": codes, "v_scales": scales}

    own, first = rows(B, S, P), rows(1, room, 0) if room else None
    each = pos if len(pos) > 1 else pos * B
    qkv = np.zeros((B, heads + 2 * kv, dim), np.float32)
    qkv[:, :heads] = r.standard_normal((B, heads, dim))
    for b, p in enumerate(each):
        if p >= 0:
            qkv[b, heads + kv:, (P + p) % dim] = r.uniform(63, 127, kv)
    cos, sin = plain.tables(S + room, dim)
    args = (dev(qkv.reshape(B, -1)), to_gpu(sgq, own))
    rest = (dev(cos), dev(sin), ints(*pos), heads)
    got = sgq.attn_decode_prefix_int8(*args, to_gpu(sgq, first), ints(P), *rest) if room else sgq.attn_decode_int8(*args, *rest)
    got = got.cpu().numpy().reshape(B, kv, heads // kv, dim)
    for b, p in enumerate(each):
        if p < 0:
            assert not got[b].any()
            continue
        n = P + p + 1
        tol = (24 + 2 * (n / 128 + 1 + 40)) * 2.0 ** -24
        for h in range(kv):
            sizes = [first["v_scales"][0, h, :P].astype(np.float64)] if P else []
            codes, scale = plain.held(qkv[b, heads + kv + h])
            assert codes[(P + p) % dim] == 127
            sizes = 127 * np.concatenate(sizes + [own["v_scales"][b, h, :p].astype(np.float64), [np.float64(scale)]])
            total = np.bincount(np.arange(n) % dim, sizes, dim)
            assert (sizes / total[np.arange(n) % dim]).min() > 4 * tol, "a lost row would not show"
            off = np.abs(got[b, h] - total / n)
            assert (off <= tol * total / n).all(), (b, h, (off / np.maximum(total / n, 1e-30)).max() / tol, np.nonzero((off > tol * total / n).any(0))[0][:8])


# ---- one value of a query far above the others ----------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("times", [30, 300, 3000])
def test_queries_with_one_large_value(sgq, form, dim, times):
    """A rotary pair of the queries `times` the others, its keys as much smaller, so that it adds to the scores what any other does.  The bound
    that the header states holds: the query's fixed point is relative to its largest value, so the score's error is too
    (tests/kv_int8_plain.py has it with max |q|), and the error is not merely that of an fp32 evaluation."""
    step = Step(form, dim, 1.0, 1.0, 1.0)
    pair = [5, 5 + dim // 2]
    step.qkv[:, :step.heads, pair] *= times
    step.qkv[:, step.heads:step.heads + step.kv, pair] /= times
    for cache in (step.own, step.first):
        if cache is not None:
            keys = cache["k_codes"].astype(np.float32) * cache["k_scales"][..., None]
            keys[..., pair] /= times
            cache["k_codes"], cache["k_scales"] = plain.held(keys)
    step.check(sgq)
    got = step.run(sgq).reshape(step.B, step.heads, dim)
    for b in range(step.B):                     # the same, per head and with what a score is made of in the place of the largest sum of all
        for h in range(step.heads):
            k, v, q = step.rows(b, h)
            e = 2.0 ** -21 * np.abs(q).max() * np.abs(k).sum(-1) / np.sqrt(dim)
            s = k @ q / np.sqrt(dim)
            w = np.exp(s - s.max())
            w /= w.sum()
            want = w @ v
            # d out = sum w (v - out) ds, and the second order of ds; 45 + 3 n / 32 roundings of weights and sums as everywhere
            room = (w * e) @ np.abs(v - want) * (1 + 2 * e.max()) + np.abs(v).max() * (45 + 3 * len(s) / 32) * 2.0 ** -24
            assert (np.abs(got[b, h] - want) <= room).all(), (b, h)


def test_rows_behind_the_position_may_change_meanwhile(sgq):
    """Caches of which a few positions are in use, while another stream writes all the rows behind them over and over."""
    r = np.random.default_rng(6)
    for B, heads, kv, S, pos in ((8, 16, 16, 640, 129), (2, 16, 2, 9000, 40), (1, 8, 2, 80000, 600)):
        host = cache_of(r.standard_normal((B, kv, S, 128)), r.standard_normal((B, kv, S, 128)))
        cache, x = to_gpu(sgq, host), dev(r.standard_normal((B, (heads + 2 * kv) * 128)).astype(np.float32))
        cos, sin = (dev(t) for t in plain.tables(S, 128))
        at, side = ints(pos), torch.cuda.Stream()
        want = sgq.attn_decode_int8(x, cache, cos, sin, at, heads)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for i in range(60):
                for t, value in ((cache.k_codes, -128), (cache.k_scales, float("nan")), (cache.v_codes, i), (cache.v_scales, float("inf"))):
                    t[:, :, pos + 1:].fill_(value)
        got = [sgq.attn_decode_int8(x, cache, cos, sin, at, heads) for _ in range(100)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
