"""The 8-bit paged cache on the GPU against tests/kv8_plain.py: storing bit by bit, attention against 64 bits, both as they are used one behind the other, in captured
graphs, and what they refuse.  Table entries that nothing may read are -1, pages that nothing may read hold codes that are no numbers.

Tolerances of attention.  u = 2^-24 is half a step of fp32.  A score is a sum of D products: off by at most (D + 8) u S, S the largest sum of |q_d k_d| of the row
(eight more roundings for the scale, the soft cap and the exponent); a weight by twice that (numerator and sum), and the weighted sum by that plus n u, all times the largest
value.  With bf16 results queries and weights may be rounded to 11 bits (2^-11 each, a rounding being off by half a step) and the result is off by 2^-8 of itself.  Those
bounds are checked number by number.  Roundings are independent of one another, so the whole result's relative error (2-norms) is far below them: 3e-3 for bf16 (2^-8 /
sqrt 3 = 2.3e-3 were every number just above a power of two), 5e-6 for fp32 (30 u)."""
import ctypes as C

import numpy as np
import pytest

import kv8_plain as P
from device_util import BF16, F32, at, dev, f32, from_dt, i32, ptr, release, size_of, zeros

pytestmark = pytest.mark.gpu
CODES = [P.INT8, P.E4M3]
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    release()


def batch(r, new, pos, B, spare=2, shuffle=True):
    """starts, tables (unused entries -1), pages of a batch whose sequences have new[s] tokens behind pos[s] others"""
    need = [(p + n + B - 1) // B for n, p in zip(new, pos)]
    pages = sum(need) + spare
    order = r.permutation(pages) if shuffle else np.arange(pages)
    tables = np.full((len(new), max(need) + 1), -1, np.int32)
    at_ = 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at_:at_ + n]
        at_ += n
    return i32(np.concatenate([[0], np.cumsum(new)])), tables, pages


def poison(cache, tables, pos, new, after):
    """codes behind the last position of every sequence (`after`: counting the new tokens) and unused pages: no numbers, scales too"""
    bad = 0x7f if cache.code == P.E4M3 else 0x55
    used = set()
    for s, row in enumerate(tables):
        n = pos[s] + (new[s] if after else 0)
        for j in range(len(row)):
            if row[j] < 0:
                continue
            used.add(int(row[j]))
            first = min(max(n - j * cache.B, 0), cache.B)
            cache.k[row[j], :, first:], cache.v[row[j], :, first:] = bad, bad
            cache.scales[row[j], :, :, (first + 15) // 16:] = np.nan
    for p in set(range(len(cache.pool))) - used:
        cache.pool[p] = 0xff


def cos_sin(n, rot, base=10000.0):
    ang = np.arange(n)[:, None] * base ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))
    return f32(np.stack([np.cos(ang), np.sin(ang)], -1))


STORE = [
    # H, G, D, Dv, page, rot, halves, new tokens, positions before them
    (4, 2, 64, 64, 16, 64, 1, [1], [0]),
    (4, 2, 64, 64, 16, 64, 0, [1], [15]),
    (4, 4, 16, 32, 16, 8, 0, [1, 1, 1], [16, 31, 5]),
    (16, 4, 128, 128, 64, 128, 1, [1, 5, 0, 37], [777, 62, 9, 130]),
    (8, 1, 256, 256, 128, 32, 1, [200, 3], [0, 126]),
    (6, 3, 80, 48, 48, 80, 0, [47, 49, 1, 0], [1, 47, 200, 0]),
    (2, 1, 96, 256, 32, 12, 1, [33, 31, 64], [15, 17, 0]),
    (3, 3, 48, 16, 16, 0, 0, [16, 15, 17], [0, 1, 15]),
    (5, 5, 112, 80, 16, 6, 1, [2] * 40, list(range(40))),
]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("case", range(len(STORE)))
@pytest.mark.parametrize("offset", [0, 1])
def test_store_is_the_formula_bit_by_bit(gpu, code, case, offset):
    """offset 1: rows whose stride and beginning are no whole 16 bytes; rows behind the last sequence and codes of other tokens stay as they were"""
    H, G, D, Dv, B, rot, halves, new, pos = STORE[case]
    r = np.random.default_rng(100 * case + code)
    starts, tables, pages = batch(r, new, pos, B)
    n, T = int(starts[-1]), int(starts[-1]) + 3
    cache = P.Cache(code, G, D, Dv, B, pages).filled(r)
    poison(cache, tables, pos, new, False)
    ld = (H + G) * D + G * Dv + 4 + offset
    x = f32(r.standard_normal((T, ld)) * np.exp(2 * r.standard_normal((T, 1))))  # some tokens far larger than those before them
    x[0, H * D:H * D + G * D] = 0                                                # a token of zeros
    x[n:] = np.nan
    cs = cos_sin(max(p + t for p, t in zip(pos, new)) + 1, rot)
    flat = np.concatenate([np.zeros(offset, np.float32), x.ravel()])
    dx, dpool, dq, before = dev(gpu, flat), dev(gpu, cache.pool), dev(gpu, np.full(T * H * D, 7.5, np.float32)), cache.pool.copy()
    q, k, v = (x[:, a:b] for a, b in ((0, H * D), (H * D, (H + G) * D), ((H + G) * D, (H + G) * D + G * Dv)))
    want = P.store(cache, q[:n].reshape(n, H, D), k[:n].reshape(n, G, D), v[:n].reshape(n, G, Dv), starts, pos, tables, rot, halves, cs, 0.37)
    base = 4 * offset
    lib = gpu.cuda_lib()
    gpu.check(lib.ggb_op_kv8_store(code, at(dx, base), at(dx, base + 4 * H * D), at(dx, base + 4 * (H + G) * D), ld, T, len(new), dev(gpu, starts).ptr, dev(gpu, i32(pos)).ptr, H, G, D,
                                   Dv, rot, halves, dev(gpu, cs).ptr if rot else None, 0.37, dev(gpu, tables).ptr, tables.shape[1], B, dpool.ptr, dq.ptr), "kv8_store")
    got = dq.download(np.float32).reshape(T, H, D)
    assert np.array_equal(got[:n].view(np.uint32), want.view(np.uint32)) and (got[n:] == 7.5).all()
    pool = dpool.download(np.uint8).reshape(cache.pool.shape)
    assert not np.array_equal(pool, before)
    same = pool == cache.pool
    assert same.all(), f"{(~same).sum()} bytes differ, first at {np.argwhere(~same)[0]}"


@pytest.mark.parametrize("code", CODES)
def test_store_of_numbers_that_are_none_and_of_extremes(gpu, code):
    G, D, B = 2, 32, 16
    r = np.random.default_rng(5)
    x = f32(r.standard_normal((16, 2 * G * D + G * D)))
    x[1, 70], x[2, 71], x[3, 72], x[5, 130] = np.nan, np.inf, -np.inf, np.nan
    x[:, 2 * G * D - 32:2 * G * D] = f32(r.uniform(-1e-38, 1e-38, (16, 32)))      # a head of tiny keys
    x[:, 2 * G * D:2 * G * D + 32] = f32(r.uniform(-3e38, 3e38, (16, 32)))        # one of huge values
    cache = P.Cache(code, G, D, D, B, 1)
    pool, q = dev(gpu, cache.pool), zeros(gpu, 16 * G * D * 4)
    P.store(cache, x[:, :G * D].reshape(16, G, D), x[:, G * D:2 * G * D].reshape(16, G, D), x[:, 2 * G * D:].reshape(16, G, D), [0, 16], [0], [[0]], 0, 0, None, 1.0)
    dx = dev(gpu, x)
    gpu.check(gpu.cuda_lib().ggb_op_kv8_store(code, dx.ptr, at(dx, 4 * G * D), at(dx, 8 * G * D), 3 * G * D, 16, 1, dev(gpu, i32([0, 16])).ptr, dev(gpu, i32([0])).ptr, G, G, D, D, 0, 0,
                                              None, 1.0, dev(gpu, i32([0])).ptr, 1, B, pool.ptr, q.ptr), "kv8_store")
    got = pool.download(np.uint8).reshape(cache.pool.shape)
    assert np.array_equal(got, cache.pool)
    assert np.isfinite(cache.scales).all() and (P.decode(code, cache.k[0, :, :16]) == P.decode(code, cache.k[0, :, :16])).all()


# ------------------------------------------------------------------------------------------------ attention
def run_attention(gpu, dt, cache, q, T, starts, pos, tables, max_new, window=0, keep=0, cap=0.0, sink=None, gate=None, scratch=True, pool=None, slack=0):
    H, D = q.shape[1:]
    lib = gpu.cuda_lib()
    pool = pool or dev(gpu, cache.pool)
    out = dev(gpu, np.full(T * H * cache.Dv * size_of(dt), 0x41, np.uint8))
    ldg = H * cache.Dv + 3
    dg = None
    if gate is not None:
        g = np.full((T, ldg), np.nan, np.float32)
        g[:len(gate), :H * cache.Dv] = gate.reshape(len(gate), -1)
        dg = dev(gpu, g)
    nbytes = int(lib.ggb_kv8_attn_scratch_bytes(cache.Dv))
    ds = zeros(gpu, nbytes + 256) if scratch else None
    qt = np.full((T, H, D), np.nan, np.float32)
    qt[:len(q)] = q
    flat = np.concatenate([np.zeros(slack, np.float32), qt.ravel()])
    gpu.check(lib.ggb_op_kv8_attn(dt, cache.code, at(dev(gpu, flat), 4 * slack), pool.ptr, dev(gpu, i32(tables)).ptr, tables.shape[1], cache.B, T, max_new, len(pos), dev(gpu, i32(starts)).ptr,
                                  dev(gpu, i32(pos)).ptr, H, cache.G, D, cache.Dv, window, keep, cap, dev(gpu, f32(sink)).ptr if sink is not None else None, ptr(dg), ldg, out.ptr, ptr(ds),
                                  nbytes if scratch else 0), "kv8_attn")
    raw = out.download(np.uint8).reshape(T, -1)
    assert (raw[int(starts[-1]):] == 0x41).all(), "rows behind the last sequence"
    return from_dt(dt, out, (T, H, cache.Dv))[:int(starts[-1])]


def check_attention(dt, got, want, reach, D, n):
    S, V = reach[..., :1], reach[..., 1:]
    tol = (2 * (D + 8) * S + n + 64) * U * V
    if dt == BF16:
        tol = tol + (2 * S + 1) * 2.0 ** -11 * V + 2.0 ** -8 * np.abs(want)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} out of bounds, first {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert rel < (3e-3 if dt == BF16 else 5e-6), rel


ATTN = [
    # H, G, D, Dv, page, new, pos, window, keep, cap, sink, gate
    (1, 1, 16, 16, 16, [1], [0], 0, 0, 0.0, 0, 0),
    (4, 4, 64, 64, 64, [1], [63], 0, 0, 0.0, 0, 0),
    (8, 1, 128, 128, 64, [1], [64], 0, 0, 0.0, 1, 0),
    (16, 4, 128, 128, 64, [1, 1, 1, 1], [777, 0, 127, 1500], 0, 0, 0.0, 0, 0),
    (32, 2, 96, 64, 48, [1, 5, 0, 3], [300, 129, 7, 46], 0, 0, 30.0, 0, 1),
    (12, 4, 80, 112, 16, [2, 7], [15, 260], 100, 0, 0.0, 0, 0),
    (6, 6, 32, 256, 32, [4, 1], [500, 333], 65, 4, 5.0, 1, 1),
    (8, 2, 192, 48, 112, [1, 9], [1000, 3], 1, 17, 0.0, 0, 0),
    (8, 1, 256, 256, 128, [1, 2], [3001, 40], 0, 0, 0.0, 0, 0),
    (20, 5, 64, 128, 16, [3], [31], 16, 16, 0.0, 1, 0),
    (48, 1, 64, 64, 64, [1], [200], 0, 0, 0.0, 0, 0),
    (130, 1, 128, 64, 64, [1, 2], [200, 100], 0, 0, 0.0, 0, 0),
    (2, 2, 128, 128, 64, [40], [0], 0, 0, 0.0, 0, 0),
    (8, 2, 128, 128, 64, [65, 1, 0, 100], [30, 90, 0, 0], 0, 0, 0.0, 1, 1),
    (8, 2, 64, 64, 48, [150], [333], 50, 10, 30.0, 0, 0),
    (4, 1, 112, 96, 16, [129, 1, 33], [1, 400, 64], 128, 3, 0.0, 0, 1),
    (4, 2, 256, 256, 64, [50, 1], [70, 10], 0, 0, 0.0, 0, 0),
    (16, 16, 16, 16, 16, [70], [9], 33, 0, 0.0, 1, 0),
]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(gpu, dt, code, case):
    H, G, D, Dv, B, new, pos, window, keep, cap, sink, gate = ATTN[case]
    r = np.random.default_rng(1000 + 10 * case + code)
    starts, tables, pages = batch(r, new, pos, B)
    cache = P.Cache(code, G, D, Dv, B, pages).filled(r)
    poison(cache, tables, pos, new, True)
    n = int(starts[-1])
    q = f32(r.standard_normal((n, H, D)) * 1.5 * D ** -0.5)
    sk = f32(r.standard_normal(H)) if sink else None
    gt = f32(2 * r.standard_normal((n, H, Dv))) if gate else None
    if window > 0:  # what lies behind every window has gone back to the pool
        for s in range(len(new)):
            for j in range(tables.shape[1]):
                if (j + 1) * B <= pos[s] - window + 1 and j * B >= keep:
                    tables[s, j] = -1
    full = np.where(tables < 0, 0, tables)
    want, reach = P.attention(cache, q, starts, pos, full, window, keep, cap, sk, gt)
    longest = max(p + t for p, t in zip(pos, new))
    for scratch in (True, False):
        got = run_attention(gpu, dt, cache, q, n + 2, starts, pos, tables, max(new), window, keep, cap, sk, gt, scratch)
        check_attention(dt, got, want, reach, D, longest)
    got = run_attention(gpu, dt, cache, q, n + 2, starts, pos, tables, n + 2, window, keep, cap, sk, gt, True, slack=1)  # queries off the 16 bytes; a bound on the tokens far too large
    check_attention(dt, got, want, reach, D, longest)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
def test_attention_is_the_same_bits_again(gpu, dt, code):
    r = np.random.default_rng(3)
    new, pos = [1, 3, 50, 1], [4000, 900, 100, 0]
    starts, tables, pages = batch(r, new, pos, 64)
    cache = P.Cache(code, 2, 128, 128, 64, pages).filled(r)
    q = f32(r.standard_normal((int(starts[-1]), 8, 128)) * 0.2)
    pool = dev(gpu, cache.pool)
    first = run_attention(gpu, dt, cache, q, len(q), starts, pos, tables, 50, pool=pool)
    for _ in range(5):
        assert np.array_equal(run_attention(gpu, dt, cache, q, len(q), starts, pos, tables, 50, pool=pool), first)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T", [1, 40])
def test_attention_where_one_key_has_all_the_weight(gpu, dt, T):
    """scores far apart, as no soft-max may overflow by; keys of zeros, whose scale is 0; values of very different scales"""
    r = np.random.default_rng(4)
    G, D, B, pos = 2, 64, 16, [200]
    starts, tables, pages = batch(r, [T], pos, B)
    cache = P.Cache(P.INT8, G, D, D, B, pages).filled(r)
    cache.k[tables[0, 2]], cache.scales[tables[0, 2], :, 0] = 0, 0
    cache.v[tables[0, 3]], cache.scales[tables[0, 3], :, 1] = 0, 0
    cache.scales[tables[0, 4], :, 1] *= np.float32(1e-30)
    cache.scales[tables[0, 5], :, 1] *= np.float32(1e20)
    q = f32(r.standard_normal((T, 4, D)) * 20)
    q[0, 1] = 0  # every key the same weight
    q[T - 1, 2] *= np.float32(1e-30)
    want, reach = P.attention(cache, q, starts, pos, tables)
    got = run_attention(gpu, dt, cache, q, T, starts, pos, tables, T)
    S, V = reach[..., :1], reach[..., 1:]
    # the largest values are 1e20 times the others: bounds are relative to them
    tol = (2 * (D + 8) * S + 600) * U * V + ((2 * S + 1) * 2.0 ** -11 * V + 2.0 ** -8 * np.abs(want) if dt == BF16 else 0)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("T", [1, 64])
def test_a_query_that_is_no_number_spoils_its_own_row_only(gpu, T):
    r = np.random.default_rng(6)
    starts, tables, pages = batch(r, [T, 2], [100, 30], 64)
    cache = P.Cache(P.INT8, 1, 64, 64, 64, pages).filled(r)
    q = f32(r.standard_normal((T + 2, 2, 64)) * 0.2)
    want, reach = P.attention(cache, q, starts, [100, 30], tables)
    q[0, 0, 5], q[T, 1, 9] = np.nan, np.nan
    got = run_attention(gpu, F32, cache, q, T + 2, starts, [100, 30], tables, T)
    for t, h in ((0, 0), (T, 1)):
        assert np.isnan(got[t, h]).all()
        got[t, h], want[t, h] = 0, 0
    check_attention(F32, got, want, reach, 64, 200)


def test_pages_beyond_32_bits(gpu):
    """a pool of more than 4 GiB: pages at both ends of it"""
    lib = gpu.cuda_lib()
    G, D, B, code = 8, 128, 64, P.INT8
    page = int(lib.ggb_kv8_page_bytes(G, D, D, B))
    pages = (1 << 32) // page + 64
    pool = gpu.DeviceBuffer(pages * page)
    r = np.random.default_rng(7)
    new, pos = [20, 1], [50, 100]
    starts, small, n_small = batch(r, new, pos, B, 0, False)
    cache = P.Cache(code, G, D, D, B, n_small).filled(r)
    far = np.array([0, pages - 1, pages // 2 + 1, pages - 7, 3, pages - 2])[:n_small]
    tables = np.where(small < 0, -1, far[np.maximum(small, 0)]).astype(np.int32)
    for i, p in enumerate(far):
        a = np.ascontiguousarray(cache.pool[i])
        gpu.check(lib.ggb_upload(pool.ptr.value + int(p) * page, a.ctypes.data_as(C.c_void_p), a.nbytes), "upload")
        gpu.sync()
    T, H = 21, 16
    x = f32(r.standard_normal((T, (H + 2 * G) * D)))
    cs = cos_sin(128, D)
    dx, dq, ds, dp, dt_ = dev(gpu, x), zeros(gpu, T * H * D * 4), dev(gpu, starts), dev(gpu, i32(pos)), dev(gpu, tables)
    qw = P.store(cache, x[:, :H * D].reshape(T, H, D), x[:, H * D:(H + G) * D].reshape(T, G, D), x[:, (H + G) * D:].reshape(T, G, D), starts, pos, small, D, 1, cs, D ** -0.5)
    gpu.check(lib.ggb_op_kv8_store(code, dx.ptr, at(dx, 4 * H * D), at(dx, 4 * (H + G) * D), x.shape[1], T, 2, ds.ptr, dp.ptr, H, G, D, D, D, 1, dev(gpu, cs).ptr, D ** -0.5, dt_.ptr,
                                   tables.shape[1], B, pool.ptr, dq.ptr), "kv8_store")
    got = np.empty(page, np.uint8)
    for i, p in enumerate(far):
        gpu.check(lib.ggb_download(got.ctypes.data_as(C.c_void_p), pool.ptr.value + int(p) * page, page), "download")
        assert np.array_equal(got, cache.pool[i].ravel())
    want, reach = P.attention(cache, qw, starts, pos, small)
    check_attention(F32, run_attention(gpu, F32, cache, qw, T, starts, pos, tables, 20, pool=pool), want, reach, D, 101)
    pool.free()


# ------------------------------------------------------------------------------------------------ as they are used
def test_a_batch_served_token_by_token_and_in_portions(gpu):
    """three sequences grow by portions and single tokens, drop tokens again and end; after every step the cache and the results are the plain form's.  Every
    step is one captured graph per shape, replayed with other starts, positions and tables"""
    lib, r = gpu.cuda_lib(), np.random.default_rng(8)
    code, H, G, D, B, n_seq, T = P.E4M3, 8, 2, 64, 16, 3, 48
    pages = 40
    free = list(r.permutation(pages))
    cache = P.Cache(code, G, D, D, B, pages)
    tables = np.full((n_seq, 16), -1, np.int32)
    cs = cos_sin(256, D)
    dx, dpool, dq, dout = zeros(gpu, T * (H + 2 * G) * D * 4), dev(gpu, cache.pool), zeros(gpu, T * H * D * 4), zeros(gpu, T * H * D * 4)
    dstarts, dpos, dtables, dcs = zeros(gpu, 4 * (n_seq + 1)), zeros(gpu, 4 * n_seq), zeros(gpu, tables.nbytes), dev(gpu, cs)
    nbytes = int(lib.ggb_kv8_attn_scratch_bytes(D))
    scratch = zeros(gpu, nbytes)
    ld = (H + 2 * G) * D

    def calls():
        gpu.check(lib.ggb_op_kv8_store(code, dx.ptr, at(dx, 4 * H * D), at(dx, 4 * (H + G) * D), ld, T, n_seq, dstarts.ptr, dpos.ptr, H, G, D, D, D, 0, dcs.ptr, 0.125, dtables.ptr, 16, B,
                                       dpool.ptr, dq.ptr), "kv8_store")
        gpu.check(lib.ggb_op_kv8_attn(F32, code, dq.ptr, dpool.ptr, dtables.ptr, 16, B, T, T, n_seq, dstarts.ptr, dpos.ptr, H, G, D, D, 0, 0, 0.0, None, None, 0, dout.ptr, scratch.ptr,
                                      nbytes), "kv8_attn")

    graph = None
    lens = [0, 0, 0]
    steps = [([20, 7, 0], None), ([1, 1, 17], None), ([1, 5, 1], None), ([4, 0, 1], [18, None, None]), ([1, 40, 3], None), ([0, 0, 0], None), ([3, 3, 33], [None, 2, 9])]
    for new, back in steps:
        for s in range(n_seq):
            if back and back[s] is not None:
                lens[s] = back[s]
            while (tables[s] >= 0).sum() * B < lens[s] + new[s]:
                tables[s, (tables[s] >= 0).sum()] = free.pop()
        starts = i32(np.concatenate([[0], np.cumsum(new)]))
        n = int(starts[-1])
        x = f32(r.standard_normal((T, ld)))
        for b, a in ((dx, x), (dstarts, starts), (dpos, i32(lens)), (dtables, tables)):
            b.upload(a)
        if graph is None:
            calls()  # once plainly: what a capture may not allocate
            gpu.sync()
            dpool.upload(cache.pool)
            g = C.c_void_p()
            gpu.check(lib.ggb_capture_begin(), "capture")
            calls()
            gpu.check(lib.ggb_capture_end(C.byref(g)), "capture")
            graph = g
        gpu.check(lib.ggb_graph_launch(graph), "launch")
        gpu.sync()
        qw = P.store(cache, x[:n, :H * D].reshape(n, H, D), x[:n, H * D:(H + G) * D].reshape(n, G, D), x[:n, (H + G) * D:].reshape(n, G, D), starts, lens, tables, D, 0, cs, 0.125)
        assert np.array_equal(dpool.download(np.uint8).reshape(cache.pool.shape), cache.pool)
        if n:
            want, reach = P.attention(cache, qw, starts, lens, tables)
            check_attention(F32, dout.download(np.float32).reshape(T, H, D)[:n].astype(np.float64), want, reach, D, 256)
        lens = [a + b for a, b in zip(lens, new)]
    gpu.check(lib.ggb_graph_free(graph), "free")


# ------------------------------------------------------------------------------------------------ refusals
def test_what_is_refused(gpu):
    """by the host, ahead of any launch"""
    lib, b = gpu.cuda_lib(), zeros(gpu, 1 << 20)
    p = b.ptr.value
    store = dict(code=1, q=p, k=p, v=p, ld=256, T=1, n_seq=1, starts=p, pos0=p, H=4, G=2, D=64, Dv=64, rot=64, halves=0, cs=p, scale=1.0, tables=p, table_ld=1, B=16, cache=p, q_out=p)
    for bad in (dict(code=0), dict(code=3), dict(q=None), dict(k=None), dict(v=None), dict(starts=None), dict(pos0=None), dict(tables=None), dict(cache=None), dict(q_out=None), dict(T=0),
                dict(T=-1), dict(n_seq=0), dict(H=3), dict(G=0), dict(H=0), dict(D=72), dict(Dv=8), dict(D=272), dict(Dv=0), dict(rot=65), dict(rot=66), dict(rot=-2), dict(halves=2),
                dict(cs=None), dict(ld=255), dict(table_ld=0), dict(B=24), dict(B=0), dict(cache=p + 8), dict(T=1 << 25), dict(T=1 << 24, G=4096, H=4096, ld=1 << 20)):
        assert lib.ggb_op_kv8_store(*{**store, **bad}.values()) == -2, bad
        assert b"kv8_store" in lib.ggb_last_error()
    need = int(lib.ggb_kv8_attn_scratch_bytes(64))
    attn = dict(dt=0, code=1, q=p, cache=p, tables=p, table_ld=1, B=16, T=1, max_new=1, n_seq=1, starts=p, pos0=p, H=4, G=2, D=64, Dv=64, window=0, keep=0, cap=0.0, sink=None, gate=None,
                ldg=0, out=p, scratch=None, nbytes=0)
    for bad in (dict(dt=1), dict(dt=2), dict(code=0), dict(q=None), dict(cache=None), dict(tables=None), dict(starts=None), dict(pos0=None), dict(out=None), dict(T=0), dict(max_new=0),
                dict(max_new=2), dict(n_seq=0), dict(H=5), dict(D=40), dict(Dv=264), dict(D=512), dict(B=8), dict(keep=-1), dict(cap=-1.0), dict(gate=p, ldg=255), dict(cache=p + 4),
                dict(table_ld=0), dict(cap=float("nan")), dict(scratch=p, nbytes=need - 1), dict(scratch=p + 4, nbytes=need)):
        assert lib.ggb_op_kv8_attn(*{**attn, **bad}.values()) == -2, bad
        assert b"kv8_attn" in lib.ggb_last_error()
