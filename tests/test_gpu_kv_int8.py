"""The INT8 key/value cache (include/sgq_decoder.h) against plain host forms: codes, scales and rotated queries bit for bit,
the attention in 64 bits with the bound that tests/kv_int8_plain.py derives."""
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


def random_cache(r, B, kv, S, dim, junk_from=None):
    """Quantized N(0, 1.3) rows; rows at positions junk_from[b] and behind hold the worst there is."""
    c = {}
    for name in "kv":
        c[name + "_codes"], c[name + "_scales"] = plain.held((r.standard_normal((B, kv, S, dim)) * 1.3).astype(np.float32))
        if junk_from is not None:
            for b in range(B):
                j = max(int(junk_from[b]), 0)
                c[name + "_codes"][b, :, j:] = -128
                c[name + "_scales"][b, :, j::2] = np.nan
                c[name + "_scales"][b, :, j + 1::2] = np.inf
    return c


def to_gpu(sgq, c):
    return sgq.KVCacheInt8(**{k: dev(v) for k, v in c.items()})


def to_host(cache):
    return {k: getattr(cache, k).cpu().numpy() for k in ("k_codes", "k_scales", "v_codes", "v_scales")}


def same_bits(got, want):
    for k in want:
        np.testing.assert_array_equal(got[k].view(np.uint8), want[k].view(np.uint8), err_msg=k)


# ---- write ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,T,heads,kv,dim,S,pos,n_new,offset,in_place", [
    (1, 1, 1, 1, 128, 1, [0], None, None, False),
    (2, 5, 4, 2, 64, 16, [3, 9], None, None, False),
    (3, 7, 6, 3, 128, 21, [0, 14, 20], [7, 2, 5], None, False),      # the last sequence runs out of cache
    (2, 4, 16, 16, 8, 9, [5], None, [30], True),                     # one position for all, behind a prefix
    (2, 3, 5, 1, 24, 6, [-1, 2], [3, 0], None, True),                # a position below zero; a sequence without tokens
    (1, 130, 8, 4, 256, 140, [6], None, None, False),
    (2, 6, 2, 2, 96, 12, [1, 2], [6, 4], [38], False),               # rotations that leave the tables
    (1, 33, 40, 40, 32, 64, [31], None, None, False),
])
def test_store_writes_the_quantizers_bits(sgq, B, T, heads, kv, dim, S, pos, n_new, offset, in_place):
    r = np.random.default_rng(B * 1000 + T * 10 + dim)
    rows = 48
    rows = max(rows, S)
    cos, sin = plain.tables(rows, dim)
    qkv = (r.standard_normal((B, T, heads + 2 * kv, dim)) * np.exp(2 * r.standard_normal((B, T, heads + 2 * kv, 1)))).astype(np.float32)
    qkv[0, 0, -1, : dim // 2] = 0.0
    start = {"k_codes": np.full((B, kv, S, dim), 77, np.int8), "k_scales": np.full((B, kv, S), 7.0, np.float32),
             "v_codes": np.full((B, kv, S, dim), -77, np.int8), "v_scales": np.full((B, kv, S), -7.0, np.float32)}
    want, q_want = {k: v.copy() for k, v in start.items()}, np.full((B, T, heads, dim), 5.0, np.float32)
    if in_place:
        q_want = qkv[:, :, :heads].copy()
    for b in range(B):
        for i in range(T):
            p = (pos[b] if len(pos) > 1 else pos[0]) + i
            turn = p + (offset[0] if offset else 0)
            if not 0 <= p < S or not 0 <= turn < rows or (n_new and i >= n_new[b]):
                continue
            q_want[b, i] = plain.turned(qkv[b, i, :heads], cos[turn], sin[turn])
            want["k_codes"][b, :, p], want["k_scales"][b, :, p] = plain.held(plain.turned(qkv[b, i, heads:heads + kv], cos[turn], sin[turn]))
            want["v_codes"][b, :, p], want["v_scales"][b, :, p] = plain.held(qkv[b, i, heads + kv:])
    cache, x = to_gpu(sgq, start), dev(qkv.reshape(B, T, -1))
    q_out = None if in_place else torch.full((B, T, heads * dim), 5.0, device="cuda")
    got = sgq.rope_kv_store_int8(x, cache, dev(cos), dev(sin), ints(*pos), heads, q_out=q_out, n_new=ints(*n_new) if n_new else None,
                                 rope_offset=ints(*offset) if offset else None)
    assert got is (x if in_place else q_out)
    same_bits(to_host(cache), want)
    after = x.cpu().numpy().reshape(qkv.shape)
    np.testing.assert_array_equal(after[:, :, :heads] if in_place else q_out.cpu().numpy().reshape(q_want.shape), q_want)
    np.testing.assert_array_equal(after if not in_place else after[:, :, heads:], qkv if not in_place else qkv[:, :, heads:])


def test_stored_values_are_the_packages_own_rows(sgq, port):
    """Value rows with NaN, infinities, zeros, vanishing and huge values: the codes and scales of quantize_int8 per row."""
    import oracle
    r = np.random.default_rng(3)
    dim, T = 64, 12
    v = r.standard_normal((T, dim)).astype(np.float32)
    v[1] = 0.0
    v[2] *= 1e-30
    v[3] *= 1e37
    v[4, 5] = np.nan
    v[5, 7] = np.inf
    v[6, 1], v[6, 2] = -np.inf, np.nan
    v[7] = np.nan
    v[8] = 1e-9
    v[9] = np.where(np.arange(dim) % 2, 1e-45, -1e-45)
    v[10, :8] = np.array([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 127.0], np.float32)      # ties: away from zero
    v[10, 8:] = 0.0
    qkv = np.zeros((1, T, 3, dim), np.float32)
    qkv[0, :, 2] = v
    cache = sgq.KVCacheInt8.empty(1, 1, T, dim, "cuda")
    cos, sin = (dev(t) for t in plain.tables(T, dim))
    sgq.rope_kv_store_int8(dev(qkv.reshape(1, T, -1)), cache, cos, sin, ints(0), 1)
    codes, scales = port.quantize_int8(v, oracle.PER_ROW)
    got = to_host(cache)
    np.testing.assert_array_equal(got["v_codes"][0, 0], codes.reshape(T, dim))
    assert got["v_scales"][0, 0].tobytes() == scales.tobytes()
    q = sgq.quantize_int8(dev(v), sgq.PER_ROW)
    np.testing.assert_array_equal(got["v_codes"][0, 0], q.qdata.cpu().numpy())
    assert got["v_scales"][0, 0].tobytes() == q.scales.cpu().numpy().tobytes()


def test_store_reads_rows_that_are_slices_of_wider_ones(sgq):
    r = np.random.default_rng(8)
    B, T, heads, kv, dim, S = 2, 3, 2, 1, 64, 8
    width = (heads + 2 * kv) * dim
    wide = dev(r.standard_normal((B, T, width + 36)).astype(np.float32))
    cos, sin = (dev(t) for t in plain.tables(S, dim))
    results = []
    for x in (wide[:, :, 4:4 + width], wide[:, :, 4:4 + width].contiguous(), wide[:, :, 4:4 + width].double(),
              wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :, 4:4 + width]):
        cache, q = sgq.KVCacheInt8.empty(B, kv, S, dim, "cuda"), torch.zeros(B, T, heads * dim + 4, device="cuda")
        sgq.rope_kv_store_int8(x, cache, cos, sin, ints(2, 4), heads, q_out=q[:, :, :heads * dim])
        assert not q[:, :, heads * dim:].any()
        results.append({**to_host(cache), "q": q.cpu().numpy()})
    for other in results[1:]:
        same_bits(other, results[0])


@pytest.mark.parametrize("dim", [16, 32, 64, 128, 208, 256])
def test_store_and_load_off_the_32_byte_grid(sgq, dim):
    """Rows, tables and outputs that start 16 bytes behind a multiple of 32: the bits of the aligned ones."""
    r = np.random.default_rng(dim)
    B, T, heads, kv, S = 2, 9, 3, 3, 12
    x = dev(r.standard_normal((B, T, (heads + 2 * kv) * dim)).astype(np.float32))
    cos, sin = (dev(t) for t in plain.tables(S, dim))

    def off(t):
        o = torch.empty(t.numel() + 8, device="cuda")
        return o[4 if o.data_ptr() % 32 == 0 else 8:][:t.numel()].view(t.shape).copy_(t)

    results = []
    for f in (lambda t: t, off):
        cache, q = sgq.KVCacheInt8.empty(B, kv, S, dim, "cuda"), f(torch.zeros(B, T, heads * dim, device="cuda"))
        sgq.rope_kv_store_int8(f(x), cache, f(cos), f(sin), ints(0, 3), heads, q_out=q)
        k, v = (f(torch.zeros(B, kv, S, dim, device="cuda")) for _ in range(2))
        assert (k.data_ptr() % 32 == 0) == (f is not off)
        sgq.kv_load_int8(cache, S, k_out=k, v_out=v)
        results.append({**to_host(cache), "q": q.cpu().numpy(), "k": k.cpu().numpy(), "v": v.cpu().numpy()})
    same_bits(results[1], results[0])


# ---- read back ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,batch,kv,dim,S,rows,row0,out_rows", [
    (1, 1, 1, 128, 1, 1, 0, 1), (2, 2, 3, 64, 37, 33, 0, 33), (1, 5, 2, 128, 70, 65, 0, 65), (3, 3, 2, 8, 300, 299, 7, 310),
    (1, 1, 1, 256, 5, 0, 0, 4), (2, 2, 5, 24, 1100, 1100, 0, 1100), (1, 3, 16, 128, 640, 512, 11, 640)])
def test_load_gives_code_times_scale(sgq, B, batch, kv, dim, S, rows, row0, out_rows):
    r = np.random.default_rng(S + rows)
    host = random_cache(r, B, kv, S, dim)
    host["k_scales"][0, 0, 0] = np.inf
    cache = to_gpu(sgq, host)
    k, v = (torch.full((batch, kv, out_rows, dim), 9.0, device="cuda") for _ in range(2))
    if row0 == 0 and out_rows == rows:
        got = sgq.kv_load_int8(cache, rows, batch=batch)
    else:
        got = sgq.kv_load_int8(cache, rows, batch=batch, k_out=k, v_out=v, row0=row0)
        assert got[0] is not None and got[0].data_ptr() == k.data_ptr() and got[1].data_ptr() == v.data_ptr()
    for name, g in zip("kv", got):
        with np.errstate(invalid="ignore"):
            want = host[name + "_codes"][:, :, :rows].astype(np.float32) * host[name + "_scales"][:, :, :rows, None]
        full = np.full((batch, kv, out_rows, dim), 9.0, np.float32)
        full[:, :, row0:row0 + rows] = want
        np.testing.assert_array_equal(g.cpu().numpy(), full if (row0 or out_rows != rows) else np.broadcast_to(want, full.shape))


# ---- decode attention -----------------------------------------------------------------------------------------------
def run_decode(sgq, B, heads, kv, dim, S, pos, prefix_len=None, prefix_max=0, seed=0, scale=1.0):
    r = np.random.default_rng(seed + B * 131 + heads * 17 + S)
    each = pos if len(pos) > 1 else pos * B
    host = random_cache(r, B, kv, S, dim, junk_from=[p if 0 <= p < S else 0 for p in each])
    qkv = (r.standard_normal((B, (heads + 2 * kv) * dim)) * scale).astype(np.float32)
    cos, sin = plain.tables(S + prefix_max, dim)
    first = random_cache(r, 1, kv, prefix_max, dim, junk_from=[min(max(prefix_len, 0), prefix_max)]) if prefix_len is not None else None
    used = 0 if prefix_len is None else min(max(prefix_len, 0), prefix_max)
    want, after, tol = plain.decode(qkv, host, cos, sin, pos, heads, first, used)
    cache, x = to_gpu(sgq, host), dev(qkv)
    nb = sgq.prepared_x_bytes(B, heads * dim)
    planes = torch.zeros(nb, dtype=torch.uint8, device="cuda") if nb else None

    def call(**kw):
        if prefix_len is None:
            return sgq.attn_decode_int8(x, cache, dev(cos), dev(sin), ints(*pos), heads, **kw)
        return sgq.attn_decode_prefix_int8(x, cache, to_gpu(sgq, first), ints(prefix_len), dev(cos), dev(sin), ints(*pos), heads, **kw)

    out = call(prepared=planes)
    again = call(out=torch.full((B, heads * dim), float("nan"), device="cuda"))     # the row is there already: nothing changes
    got = out.cpu().numpy()
    assert np.array_equal(got, again.cpu().numpy()), "the same call gives other bits"
    same_bits(to_host(cache), after)
    np.testing.assert_array_equal(x.cpu().numpy(), qkv)
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()
    if nb:
        assert torch.equal(planes, sgq.prepare_x(out, torch.zeros(nb, dtype=torch.uint8, device="cuda")))
    return got


DECODE = [
    (1, 1, 1, 128, 1, [0]), (1, 1, 1, 64, 8, [7]), (2, 2, 2, 128, 64, [6, 0]), (1, 8, 1, 128, 70, [32]), (8, 16, 16, 128, 640, [129]),
    (3, 5, 5, 64, 333, [332, 0, 31]), (2, 12, 3, 64, 100, [63, 64]), (2, 10, 2, 128, 257, [255, 256]), (1, 14, 2, 64, 1000, [999]),
    (2, 32, 4, 128, 300, [299, 150]), (1, 16, 1, 128, 90, [33]), (1, 34, 2, 64, 50, [40]), (40, 32, 32, 64, 128, [100]),
    (5, 4, 1, 128, 2051, [2050, -1, 17, 2051, 1024]), (1, 4, 2, 128, 9001, [9000]), (3, 20, 4, 128, 31, [-5, 30, 1]), (37, 8, 8, 64, 512, [500]), (33, 16, 16, 128, 300, [255]),
    (16, 8, 4, 128, 1500, [1499 - 99 * i for i in range(16)]), (9, 40, 8, 64, 700, [699, 64, 63, 128, 127, 0, 1, -1, 300])]


# caches that may grow long (dealt out to all warps of the device): few and many positions in them, idle slots at every place
LONG = [
    (1, 4, 2, 128, 80000, [70001]), (1, 16, 16, 128, 9600, [0]), (3, 6, 6, 128, 7000, [6999, 63, 64]), (2, 32, 4, 64, 20000, [127, 19999]),
    (5, 8, 8, 64, 2000, [-1, 1999, -1, 128, -1]), (2, 48, 4, 128, 19000, [300, 5000]), (37, 2, 1, 64, 5000, [500]), (2, 40, 2, 128, 16000, [15999, 0]),
    (40, 4, 1, 128, 2000, [(51 * i) % 2003 - 2 for i in range(40)]), (4, 10, 2, 128, 20000, [-1, -1, -1, -1]), (33, 1, 1, 128, 3000, [255])]


@pytest.mark.parametrize("B,heads,kv,dim,S,pos", LONG)
def test_decode_over_long_caches(sgq, B, heads, kv, dim, S, pos):
    assert sgq.lib.sgqd_attn_decode_int8_workspace_bytes(B, heads, kv, dim, S) > 0
    got = run_decode(sgq, B, heads, kv, dim, S, pos)
    for b, p in enumerate(pos if len(pos) > 1 else pos * B):
        if not 0 <= p < S:
            assert not got[b].any()


@pytest.mark.parametrize("B,heads,kv,dim,S,pos", DECODE)
def test_decode(sgq, B, heads, kv, dim, S, pos):
    got = run_decode(sgq, B, heads, kv, dim, S, pos)
    for b, p in enumerate(pos if len(pos) > 1 else pos * B):
        if not 0 <= p < S:
            assert not got[b].any()


@pytest.mark.parametrize("scale", [1e-20, 0.0, 30.0])
def test_decode_with_vanishing_and_steep_scores(sgq, scale):
    run_decode(sgq, 2, 4, 2, 128, 200, [199, 40], scale=scale)


PREFIX = [
    (1, 1, 1, 128, 4, [0], 1, 1), (2, 2, 2, 64, 16, [3, 15], 33, 40), (8, 16, 16, 128, 32, [9], 200, 256), (3, 12, 4, 64, 20, [0, 19, -1], 65, 65),
    (5, 8, 1, 128, 40, [39, 1, 2, 3, 40], 513, 600), (9, 14, 2, 128, 12, [4], 31, 64), (33, 4, 4, 64, 5, [2], 130, 130), (2, 16, 1, 64, 8, [7, 0], 3001, 3001),
    (2, 4, 2, 128, 50, [49, 12], 0, 8), (2, 4, 2, 128, 50, [49, 12], -3, 8), (2, 4, 2, 128, 50, [49, 12], 99, 8), (3, 6, 6, 128, 7000, [6999, -1, 3], 700, 720), (70, 8, 2, 128, 6, [5], 90, 90)]
# one to 130 query rows per kv head, prefixes that end inside, at and behind a tile of 32 and of 128 positions
PREFIX += [(2, 16, 2, 128, 40, [33, 2], n, 400) for n in (31, 32, 33, 127, 128, 129, 256, 257, 400)]
PREFIX += [(B, 10, 10, dim, 40, [33], 300, 384) for B in (7, 8, 9, 16, 17, 24, 32, 33, 127, 128, 129) for dim in (64, 128)]
PREFIX += [(35, 4, 2, dim, 40, [33], n, 1000) for dim in (64, 128) for n in (1, 31, 127, 128, 129, 255, 256, 1000)]
PREFIX += [(34, 1, 1, 128, 8, [2], 20011, 20480), (130, 2, 1, 64, 8, [2], 5000, 5000), (1, 7, 1, 128, 8, [2], 20011, 20480)]


@pytest.mark.parametrize("B,heads,kv,dim,S,pos,prefix_len,prefix_max", PREFIX)
def test_decode_behind_a_shared_prefix(sgq, B, heads, kv, dim, S, pos, prefix_len, prefix_max):
    got = run_decode(sgq, B, heads, kv, dim, S, pos, prefix_len, prefix_max)
    for b, p in enumerate(pos if len(pos) > 1 else pos * B):
        if not 0 <= p < S:
            assert not got[b].any()


def test_values_that_are_not_finite_reach_their_own_head_only(sgq):
    B, heads, kv, dim, S, p = 3, 4, 2, 128, 80, 70
    r = np.random.default_rng(11)
    host = random_cache(r, B, kv, S, dim)
    qkv = r.standard_normal((B, heads + 2 * kv, dim)).astype(np.float32)
    cos, sin = plain.tables(S, dim)
    clean = plain.decode(qkv.reshape(B, -1), host, cos, sin, [p], heads)
    qkv[0, 1, 5] = np.nan                          # query head 1 of sequence 0
    qkv[0, 2, 9] = -np.inf                         # query head 2 of sequence 0
    host["k_scales"][1, 0, 33] = np.inf            # heads 0 and 1 of sequence 1
    host["v_scales"][2, 1, 12] = np.inf            # heads 2 and 3 of sequence 2
    host["v_scales"][2, 0, 13] = np.nan            # heads 0 and 1 of sequence 2
    bad = {(0, 1), (0, 2), (1, 0), (1, 1), (2, 0), (2, 1), (2, 2), (2, 3)}
    cache = to_gpu(sgq, host)
    out = sgq.attn_decode_int8(dev(qkv.reshape(B, -1)), cache, dev(cos), dev(sin), ints(p), heads).cpu().numpy().reshape(B, heads, dim)
    for b in range(B):
        for h in range(heads):
            if (b, h) in bad:
                assert np.isnan(out[b, h]).all(), (b, h)
            else:
                at = slice(h * dim, (h + 1) * dim)
                assert (np.abs(out[b, h] - clean[0][b, at]) <= clean[2][b, at]).all(), (b, h)


@pytest.mark.parametrize("B", [2, 12, 40])              # 8 (mma.sync, one warp of rows), 48 and 160 query rows per kv head
@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_are_not_finite_behind_a_prefix(sgq, B, dim):
    heads, kv, S, p, P = 8, 2, 40, 30, 300
    r = np.random.default_rng(21)
    host, first = random_cache(r, B, kv, S, dim), random_cache(r, 1, kv, P + 20, dim, junk_from=[P])
    qkv = r.standard_normal((B, heads + 2 * kv, dim)).astype(np.float32)
    cos, sin = plain.tables(S + P + 20, dim)
    clean = plain.decode(qkv.reshape(B, -1), host, cos, sin, [p], heads, first, P)

    def run():
        out = sgq.attn_decode_prefix_int8(dev(qkv.reshape(B, -1)), to_gpu(sgq, host), to_gpu(sgq, first), ints(P), dev(cos), dev(sin), ints(p), heads)
        return out.cpu().numpy().reshape(B, heads, dim)

    def check(out, bad):
        for b in range(B):
            for h in range(heads):
                if bad(b, h):
                    assert np.isnan(out[b, h]).all(), (b, h)
                else:
                    at = slice(h * dim, (h + 1) * dim)
                    assert (np.abs(out[b, h] - clean[0][b, at]) <= clean[2][b, at]).all(), (b, h)

    qkv[0, 1, 5], qkv[B - 1, 6, 0] = np.nan, np.inf
    rows = {(0, 1), (B - 1, 6)}
    check(run(), lambda b, h: (b, h) in rows)
    for name, value, at in (("k_scales", np.inf, 7), ("k_scales", np.nan, 290), ("v_scales", np.inf, 150), ("v_scales", np.nan, 0)):
        kept = first[name].copy()
        first[name][0, 1, at] = value                # heads 4 to 7 of every sequence
        check(run(), lambda b, h: h >= 4 or (b, h) in rows)
        first[name][:] = kept


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("B,heads,kv,S,P", [(2, 4, 2, 400, 0), (2, 4, 1, 9600, 0), (2, 4, 2, 40, 700), (8, 4, 1, 40, 700), (12, 8, 2, 40, 700)])
def test_outputs_beside_a_token_that_takes_the_weight(sgq, B, heads, kv, S, P, dim):
    """The first token of each sequence (of the prefix, where there is one) has nearly all the weight and values of next to nothing;
    what the others leave, e^-20 times their values each, has to keep its precision: tests/kv_int8_plain.py's bound, but relative
    to sum w |v| / sum w in the place of max |v|.  The other tokens weigh the same, so a weight's fixed point, relative to the
    largest around it, is relative to the weight."""
    r = np.random.default_rng(B + S + P)
    pos = S - 7
    cos, sin = plain.tables(S + P, dim)
    q = r.standard_normal(dim).astype(np.float32)
    qkv = np.zeros((B, heads + 2 * kv, dim), np.float32)
    qkv[:, :heads] = q
    qkv[:, heads + kv:] = r.standard_normal((B, kv, dim))
    turned = plain.turned(q, cos[P + pos], sin[P + pos])
    sink = turned * np.float32(20 * np.sqrt(dim) / (turned.astype(np.float64) ** 2).sum())

    def held(batch, rows, with_sink):
        c, k = {}, np.zeros((batch, kv, rows, dim), np.float32)
        v = r.standard_normal((batch, kv, rows, dim)).astype(np.float32)
        if with_sink:
            k[:, :, 0], v[:, :, 0] = sink, v[:, :, 0] * 1e-12
        c["k_codes"], c["k_scales"] = plain.held(k)
        c["v_codes"], c["v_scales"] = plain.held(v)
        return c

    own, first = held(B, S, P == 0), held(1, P, True) if P else None
    want, _, tol = plain.decode(qkv.reshape(B, -1), own, cos, sin, [pos], heads, first, P)
    size = {}
    for name, c in (("own", own), ("first", first)):
        size[name] = None if c is None else {**c, "v_codes": np.abs(c["v_codes"])}
    positive = np.abs(qkv)
    positive[:, :heads + kv] = qkv[:, :heads + kv]
    weighed, _, _ = plain.decode(positive.reshape(B, -1), size["own"], cos, sin, [pos], heads, size["first"], P)
    most = np.zeros_like(tol)                                         # max |v|, by which tol is made
    for b in range(B):
        for h in range(heads):
            hk = h // (heads // kv)
            v = [np.abs(c["v_codes"][i, hk, :n].astype(np.float64) * c["v_scales"][i, hk, :n, None]).max()
                 for c, i, n in ((own, b, pos), (first, 0, P)) if c is not None and n] + [np.abs(plain.held(qkv[b, heads + kv + hk])[0] / 127.0).max() * np.abs(qkv[b, heads + kv + hk]).max()]
            most[b, h * dim:(h + 1) * dim] = max(v)
    args = (dev(qkv.reshape(B, -1)), to_gpu(sgq, own))
    rest = (dev(cos), dev(sin), ints(pos), heads)
    got = sgq.attn_decode_prefix_int8(*args, to_gpu(sgq, first), ints(P), *rest) if P else sgq.attn_decode_int8(*args, *rest)
    off = np.abs(got.cpu().numpy() - want) / (tol / most * weighed)
    assert (weighed < 0.02 * most).all() and off.max() <= 1, off.max()


def test_decode_and_store_hold_the_same_row(sgq):
    """A token appended by the decode step and by the prompt's store: the same bits; and the rows read back."""
    B, heads, kv, dim, S = 4, 8, 4, 128, 33
    r = np.random.default_rng(12)
    x = dev(r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32))
    cos, sin = (dev(t) for t in plain.tables(S, dim))
    pos = ints(0, 32, 5, -1)
    a, b = (sgq.KVCacheInt8.empty(B, kv, S, dim, "cuda") for _ in range(2))
    sgq.attn_decode_int8(x, a, cos, sin, pos, heads)
    sgq.rope_kv_store_int8(x[:, None].clone(), b, cos, sin, pos, heads)
    same_bits(to_host(a), to_host(b))


def test_rows_and_outputs_that_are_slices(sgq):
    B, heads, kv, dim, S = 3, 4, 2, 64, 40
    r = np.random.default_rng(13)
    host = random_cache(r, B, kv, S, dim)
    width = (heads + 2 * kv) * dim
    wide = dev(r.standard_normal((B, width + 12)).astype(np.float32))
    cos, sin = (dev(t) for t in plain.tables(S, dim))
    pos = ints(20, 39, 3)
    want = sgq.attn_decode_int8(wide[:, 4:4 + width].contiguous(), to_gpu(sgq, host), cos, sin, pos, heads)
    out = torch.full((B, heads * dim + 3), 5.0, device="cuda")
    for x in (wide[:, 4:4 + width], wide[:, 4:4 + width].unsqueeze(1), wide[:, 4:4 + width].double()):
        out.fill_(5.0)
        sgq.attn_decode_int8(x, to_gpu(sgq, host), cos, sin, pos, heads, out=out[:, 1:1 + heads * dim])
        assert torch.equal(out[:, 1:1 + heads * dim], want) and bool((out[:, 0] == 5).all()) and bool((out[:, -2:] == 5).all())
    shifted = torch.empty(B * width + 1, device="cuda")[1:].view(B, width).copy_(wide[:, 4:4 + width])       # rows off the 16-byte grid
    assert torch.equal(sgq.attn_decode_int8(shifted, to_gpu(sgq, host), cos, sin, pos, heads), want)


def test_cache_larger_than_two_gib(sgq):
    """The last sequences' rows lie behind 2^31 codes."""
    B, heads, kv, dim, S = 17, 16, 16, 128, 63000          # 2.19e9 codes
    r = np.random.default_rng(14)
    codes, scales = (torch.zeros(B, kv, S, dim, dtype=torch.int8, device="cuda") for _ in range(2)), (torch.zeros(B, kv, S, device="cuda") for _ in range(2))
    cache = sgq.KVCacheInt8(*(x for pair in zip(codes, scales) for x in pair))
    assert cache.k_codes.numel() > 2 ** 31
    small = random_cache(r, B, kv, 40, dim)
    for k, v in small.items():
        getattr(cache, k)[:, :, :40] = dev(v)
    cos, sin = plain.tables(S, dim)
    qkv = r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32)
    want, after, tol = plain.decode(qkv, small, cos, sin, [37], heads)
    out = sgq.attn_decode_int8(dev(qkv), cache, dev(cos), dev(sin), ints(37), heads).cpu().numpy()
    assert (np.abs(out - want) <= tol).all()
    same_bits({k: getattr(cache, k)[:, :, :40].cpu().numpy() for k in after}, after)
    x = dev(qkv).view(B, 1, -1)
    sgq.rope_kv_store_int8(x, cache, dev(cos), dev(sin), ints(62999), heads)
    k, v = plain.held(plain.turned(qkv[-1].reshape(-1, dim)[heads:heads + kv], cos[62999], sin[62999])), plain.held(qkv[-1].reshape(-1, dim)[heads + kv:])
    np.testing.assert_array_equal(cache.k_codes[-1, :, -1].cpu().numpy(), k[0])
    np.testing.assert_array_equal(cache.v_codes[-1, :, -1].cpu().numpy(), v[0])
    last = sgq.KVCacheInt8(*(getattr(cache, n)[-1:, -1:] for n in ("k_codes", "k_scales", "v_codes", "v_scales")))
    k_back, _ = sgq.kv_load_int8(last, S)
    np.testing.assert_array_equal(k_back[0, 0, -1].cpu().numpy(), k[0][-1].astype(np.float32) * k[1][-1])


# ---- streams, graphs ------------------------------------------------------------------------------------------------
def test_decode_steps_in_a_graph_on_a_side_stream(sgq):
    """A captured pair of decode steps (with and without a prefix, one workspace) replayed while the positions advance, next to
    the same steps run eagerly."""
    B, heads, kv, dim, S, P = 3, 8, 4, 128, 48, 100
    r = np.random.default_rng(15)
    host, first = random_cache(r, B, kv, S, dim), to_gpu(sgq, random_cache(r, 1, kv, P, dim))
    cos, sin = (dev(t) for t in plain.tables(S + P, dim))
    steps = [dev(r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32)) for _ in range(4)]
    length = ints(P)

    def eager():
        a, b, got = to_gpu(sgq, host), to_gpu(sgq, host), []
        for i, x in enumerate(steps):
            pos = ints(10 + i, i, 40 + i)
            got.append((sgq.attn_decode_int8(x, a, cos, sin, pos, heads), sgq.attn_decode_prefix_int8(x, b, first, length, cos, sin, pos, heads)))
        return got, a, b

    want, wa, wb = eager()
    a, b, ws = to_gpu(sgq, host), to_gpu(sgq, host), sgq.Workspace("cuda")
    x, pos, out_a, out_b = steps[0].clone(), ints(10, 0, 40), torch.empty(B, heads * dim, device="cuda"), torch.empty(B, heads * dim, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        warm_a, warm_b = to_gpu(sgq, host), to_gpu(sgq, host)
        sgq.attn_decode_int8(x, warm_a, cos, sin, pos, heads, out=out_a)
        sgq.attn_decode_prefix_int8(x, warm_b, first, length, cos, sin, pos, heads, out=out_b, workspace=ws)
        side.synchronize()
        graphs = []
        for _ in range(2):                       # two graphs that share the workspace, replayed in turn
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                sgq.attn_decode_int8(x, a, cos, sin, pos, heads, out=out_a)
                sgq.attn_decode_prefix_int8(x, b, first, length, cos, sin, pos, heads, out=out_b, workspace=ws)
            graphs.append(g)
        for i, step in enumerate(steps):
            x.copy_(step)
            pos.copy_(ints(10 + i, i, 40 + i))
            graphs[i % 2].replay()
            assert torch.equal(out_a, want[i][0]) and torch.equal(out_b, want[i][1]), i
        side.synchronize()
    same_bits(to_host(a), to_host(wa))
    same_bits(to_host(b), to_host(wb))
    assert sgq.device_status() == 0


def test_two_calls_at_once_on_two_streams(sgq):
    B, heads, kv, dim, S, P = 4, 20, 4, 128, 900, 2000
    r = np.random.default_rng(16)
    first = to_gpu(sgq, random_cache(r, 1, kv, P, dim))
    cos, sin = (dev(t) for t in plain.tables(S + P, dim))
    jobs = []
    for _ in range(2):
        host = random_cache(r, B, kv, S, dim)
        jobs.append((host, dev(r.standard_normal((B, (heads + 2 * kv) * dim)).astype(np.float32))))
    pos, length = ints(899, 700, 5, 64), ints(P)
    want = [sgq.attn_decode_prefix_int8(x, to_gpu(sgq, h), first, length, cos, sin, pos, heads) for h, x in jobs]
    caches, streams, out = [to_gpu(sgq, h) for h, _ in jobs], [torch.cuda.Stream() for _ in jobs], [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (_, x) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                out[i] = sgq.attn_decode_prefix_int8(x, caches[i], first, length, cos, sin, pos, heads)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_the_c_calls_reject_what_they_cannot_run(sgq):
    """On a device: refused before anything is launched, and the context stays usable."""
    c = sgq.CacheInt8(256, 256, 256, 256, 1, 1, 8, 96)
    one = C.c_void_p(256)
    assert sgq.lib.sgqd_attn_decode_int8(one, 288, 1, one, one, 8, one, 0, C.byref(c), one, 96, None, 0, None, 0, None) == 4
    cache = sgq.KVCacheInt8.empty(1, 1, 8, 96, "cuda")
    cos, sin = (dev(t) for t in plain.tables(8, 96))
    with pytest.raises(sgq.SgqError):
        sgq.attn_decode_int8(torch.zeros(1, 288, device="cuda"), cache, cos, sin, ints(0), 1)
    k, _ = sgq.kv_load_int8(cache, 8)
    assert not k.any()
