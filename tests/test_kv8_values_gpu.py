"""Attention over the 8-bit cache where groups' value scales, weights and scores lie far apart: every row by its own bound.

The plain form is in 64 bits; beside the result it gives, number by number, A = sum_j w_j |v_j| / sum_j w_j (what all terms of the result add up to) and, row by row, R = sum_j w_j s_j top /
sum_j w_j, s_j the scale of the group that value j lies in and top the largest code (what the terms could be: a code of j is off by half a step s_j anyway).

Bounds, u = 2^-24.  A score is off by at most (D + 8) u S (S: the largest sum of |q_d k_d| of the row), a weight by that and so is the denominator; sums of n terms by n u; 64 u for what is
rounded a few times each.  Weights go to the products as 16-bit numbers: one of 11 bits for bf16 results, 2^-11 of itself (a rounding is off by half a step), two for fp32 results, 2^-22; and,
being numbers of a smallest step, each by no more than 2^-32 of the largest product of a weight and a scale of its row: together n 2^-32 R.  With bf16 results queries may be rounded to steps of 2^-20 of their row's largest (a score
by 2^-20 Q, Q the largest sum of |k_d| times that), and the result is off by 2^-8 of itself.
Nothing else: no bound counts a value that the row does not see, or does not weigh."""
import numpy as np
import pytest

import kv8_plain as P
from device_util import BF16, F32, f32, release
from test_kv8_gpu import batch, run_attention

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CODES = [P.INT8, P.E4M3]


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    release()


def plain(cache, q, starts, pos, tables, window=0, keep=0):
    """float64: results, A [T][H][Dv]; R, S, Q, n [T][H][1]"""
    T, H, _ = q.shape
    out, A = np.zeros((T, H, cache.Dv)), np.zeros((T, H, cache.Dv))
    R, S, Q, n = np.zeros((4, T, H, 1))
    for s in range(len(pos)):
        t0, new, p0 = int(starts[s]), int(starts[s + 1] - starts[s]), int(pos[s])
        k, v = cache.numbers(tables[s], p0 + new)
        j = np.arange(p0 + new)
        step = cache.scales[np.asarray(tables[s])[j // cache.B], :, 1, j % cache.B // P.GROUP].astype(np.float64)
        for i in range(new):
            seen = j <= p0 + i
            if window > 0:
                seen &= (p0 + i - j < window) | (j < keep)
            for h in range(H):
                g, x = h // (H // cache.G), q[t0 + i, h].astype(np.float64)
                z = k[seen, g] @ x
                w = np.exp(z - z.max())
                w /= w.sum()
                out[t0 + i, h], A[t0 + i, h] = w @ v[seen, g], w @ np.abs(v[seen, g])
                R[t0 + i, h], S[t0 + i, h], n[t0 + i, h] = P.TOP[cache.code] * (w @ step[seen, g]), (np.abs(k[seen, g]) @ np.abs(x)).max(), seen.sum()
                Q[t0 + i, h] = np.abs(k[seen, g]).sum(1).max() * np.abs(x).max()
    return out, A, R, S, Q, n


def check(dt, got, form, D):
    out, A, R, S, Q, n = form
    tol = ((2 * (D + 8) * S + n + 64) * U + 2.0 ** -21) * A + n * 2.0 ** -32 * R
    if dt == BF16:
        tol = tol + (2.0 ** -19 * Q + 2.0 ** -11) * A
        tol = tol + 2.0 ** -8 * (np.abs(out) + tol)
    bad = ~(np.abs(got - out) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} out of bounds, first {np.argwhere(bad)[0]}: {got[bad][0]} for {out[bad][0]}, {(np.abs(got - out) / tol)[bad].max()} times the bound"


def both(gpu, dt, cache, q, starts, pos, tables, most, window=0, keep=0):
    form = plain(cache, q, starts, pos, np.maximum(tables, 0), window, keep)
    for scratch in (True, False):
        check(dt, run_attention(gpu, dt, cache, q, len(q), starts, pos, tables, most, window, keep, scratch=scratch), form, q.shape[2])


# rows of a key head: 2, 12 (steps) and 160 (a portion); heads of 64 and, steps only, 256
FORMS = [(1, 2, 64), (3, 4, 64), (40, 4, 64), (3, 4, 256)]


def made(code, T, H, D, pos, seed, spread=0.2, B=32):
    r = np.random.default_rng(seed)
    starts, tables, pages = batch(r, [T], [pos], B)
    cache = P.Cache(code, 1, D, D, B, pages).filled(r)
    return r, cache, starts, tables, f32(r.standard_normal((T, H, D)) * spread)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H,D", FORMS)
@pytest.mark.parametrize("big", [1e2, 1e5, 1e8, 1e20])
def test_large_values_of_no_weight(gpu, dt, code, T, H, D, big):
    """a page whose values are far above the others', and whose keys every query turns away: scores of -90"""
    r, cache, starts, tables, q = made(code, T, H, D, 300, 1)
    page = tables[0, 4]
    cache.scales[page, :, 1] *= np.float32(big)
    cache.k[page, 0, :, 0] = P.encode(code, np.full(cache.B, -P.TOP[code], np.float32))
    q[..., 0] = 90.0 / (P.TOP[code] * float(cache.scales[page, 0, 0].min()))
    cache.k[np.arange(len(cache.k)) != page, 0, :, 0] = 0
    both(gpu, dt, cache, q, starts, [300], tables, T)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H", [(5, 4), (40, 4), (70, 2)])
@pytest.mark.parametrize("big", [1e3, 1e6])
def test_large_values_of_later_tokens(gpu, dt, code, T, H, big):
    """what a portion's last tokens bring changes nothing for the ones before them"""
    r, cache, starts, tables, q = made(code, T, H, 64, 64 - 16 * (T == 5) - 2 * (T == 5), 2)
    pos = 46 if T == 5 else 64
    starts, tables, pages = batch(r, [T], [pos], 32)
    cache = P.Cache(code, 1, 64, 64, 32, pages).filled(r)
    last = pos + T - 1
    for first in range(last - last % 16 - (16 if T > 40 else 0), last + 1, 16):
        cache.scales[tables[0, first // 32], :, 1, first % 32 // 16] *= np.float32(big)
    both(gpu, dt, cache, q, starts, [pos], tables, T)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H", [(4, 4), (40, 4)])
@pytest.mark.parametrize("big", [1e3, 1e6])
def test_large_values_outside_of_the_window(gpu, dt, code, T, H, big):
    """positions that some rows of an item see and the later ones no longer"""
    r, cache, starts, tables, q = made(code, T, H, 64, 110, 3)
    window = 33
    first = (110 - window + 1) // 16 * 16
    cache.scales[tables[0, first // 32], :, 1, first % 32 // 16] *= np.float32(big)
    both(gpu, dt, cache, q, starts, [110], tables, T, window, 3)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H", [(1, 4), (40, 4)])
@pytest.mark.parametrize("below", [25.5, 28.0])
def test_many_small_weights_beside_a_large_one(gpu, dt, code, T, H, below):
    """12,000 weights of 2^-25.5 (2^-28) of the largest, whose own value is zero: the result is theirs"""
    r, cache, starts, tables, q = made(code, T, H, 64, 12000, 4, B=128)
    cache.k[...], cache.scales[:, :, 0] = 0, 1 / 64
    top = P.TOP[code]
    at = int(tables[0, 37])
    cache.k[at, 0, 5, 0] = P.encode(code, np.full(1, 64, np.float32))[0]  # a key of 1 along the first coordinate
    cache.v[at, 0, 5] = 0
    cache.v[...] = np.where(np.isin(cache.v, [0, 128]), cache.v, P.encode(code, np.full(1, top / 2, np.float32))[0])
    cache.v[at, 0, 5] = 0
    q[...] = 0
    q[..., 0] = below * np.log(2)
    both(gpu, dt, cache, q, starts, [12000], tables, T)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H,D", FORMS)
@pytest.mark.parametrize("kind", ["mixed", "rising", "falling", "edges"])
def test_scales_far_apart(gpu, dt, code, T, H, D, kind):
    """value scales over 17 powers of ten, along the positions or in no order; or groups of scale 0, 1e-30 and 1e20 beside ordinary ones"""
    r, cache, starts, tables, q = made(code, T, H, D, 400, 5, 0.6)
    n = tables.shape[1] * 2
    e = {"mixed": r.uniform(-9, 8, n), "rising": np.linspace(-9, 8, n), "falling": np.linspace(8, -9, n), "edges": r.choice([0.0, 0.0, -30.0, 20.0], n)}[kind]
    for j in range(n):
        if tables[0, j // 2] >= 0:
            cache.scales[tables[0, j // 2], :, 1, j % 2] *= np.float32(10.0 ** e[j] if kind != "edges" or j % 5 else 0)
            if kind == "edges" and j % 5 == 0:
                cache.v[tables[0, j // 2], :, 16 * (j % 2):16 * (j % 2) + 16] = 0
    both(gpu, dt, cache, q, starts, [400], tables, T)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,H", [(1, 4), (3, 4), (40, 4)])
@pytest.mark.parametrize("score", [5, 40, 80])
def test_equal_scores_along_different_numbers(gpu, dt, code, T, H, score):
    """two halves of the keys with the same large score, one by numbers of the query that 11 bits cut, the other by numbers that they hold, and values of either sign: what is cut off a
    query a score multiplies"""
    D = 64
    r, cache, starts, tables, q = made(code, T, H, D, 64, 6)
    top = P.TOP[code]
    cache.k[...], cache.scales[:, :, 0] = 0, 1.0
    cache.v[...], cache.scales[:, :, 1] = P.encode(code, np.full(1, top, np.float32))[0], 1 / top
    one = P.encode(code, np.full(1, 1, np.float32))[0]
    for j in range(64 + T):
        page, row = tables[0, j // 32], j % 32
        cache.k[page, 0, row, :32 if j % 2 else 0] = one
        cache.k[page, 0, row, 32:(32 if j % 2 else 64)] = one
        if j % 2:
            cache.v[page, 0, row] = P.encode(code, np.full(1, -top / 2, np.float32))[0]
    q[...] = score / 32
    q[..., :32] *= np.float32(1 + 2.0 ** -11 * 0.99)
    both(gpu, dt, cache, q, starts, [64], tables, T)
