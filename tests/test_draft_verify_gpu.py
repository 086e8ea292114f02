"""Checked drafts on the GPU against tests/kv8_plain.py.  Decisions are whole numbers: they are the plain form's wherever its nearest decision is further off than what
fp32 exponentials can move, and otherwise (the borders of a running sum over a whole vocabulary lie closer than that) within what they can move.  An exponential of (l - m)
/ t is off by 4 steps of 2^-24 (the unit's 2^-22) and by (l - m) / t times the three roundings of its argument (difference, constant, product), 2^-24 each; sums of many are
nearer than one.  Weights below e^-20 of the largest move nothing here (256,000 of them are 5e-4 of it, off by 1e-5), so that is under 64 * 2^-24 = 4e-6 of itself."""
import ctypes as C

import numpy as np
import pytest

import kv8_plain as P
from device_util import at, dev, f32, i32, release, zeros

pytestmark = pytest.mark.gpu
NEAR = 4e-6


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    release()


def run(gpu, target, draft, starts, drafted, u, t, R=None, ld=None, slack=0):
    lib = gpu.cuda_lib()
    n, V = len(starts) - 1, target.shape[1]
    R = R or len(target)
    ld = ld or V

    def rows(x):
        y = np.full(slack + R * ld, np.nan, np.float32)
        for i in range(len(x)):
            y[slack + i * ld:slack + i * ld + V] = x[i]
        return at(dev(gpu, y), 4 * slack)
    tokens, accepted = dev(gpu, np.full(R, -2, np.int32)), dev(gpu, np.full(n, -2, np.int32))
    nbytes = int(lib.ggb_draft_verify_scratch_bytes(R, n))
    scratch = dev(gpu, np.full(nbytes, 0xff, np.uint8))
    pad = lambda x, ty: np.concatenate([np.asarray(x, ty), np.zeros(R - len(x), ty)])  # noqa: E731
    for _ in range(2):  # the second time on what the first left in the workspace
        gpu.check(lib.ggb_op_draft_verify(rows(target), ld, rows(draft) if draft is not None else None, ld, V, R, n, dev(gpu, i32(starts)).ptr, dev(gpu, pad(drafted, np.int32)).ptr,
                                          dev(gpu, pad(u, np.float32)).ptr, t, tokens.ptr, accepted.ptr, scratch.ptr, nbytes), "draft_verify")
    return tokens.download(np.int32), accepted.download(np.int32)


def inputs(r, rows, V, spread=2.5):
    R = sum(rows)
    target = f32(r.standard_normal((R, V)) * spread)
    draft = f32(target + r.standard_normal((R, V)) * 0.7)
    return target, draft, i32(np.concatenate([[0], np.cumsum(rows)])), f32(r.random(R))


CASES = [([1], 1), ([1], 7), ([2], 3), ([5], 1000), ([3, 1, 6, 0, 2], 4097), ([9, 9], 2048), ([4] * 33, 50), ([2, 0, 0, 3], 32003), ([6], 256000), ([40], 301)]


@pytest.mark.parametrize("t", [1.0, 0.5, 1.7, 0.0])
@pytest.mark.parametrize("point", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_plain_form(gpu, case, t, point):
    rows, V = CASES[case]
    r = np.random.default_rng(20 + case)
    target, draft, starts, u = inputs(r, rows, V)
    noise = -np.log(-np.log(r.uniform(1e-9, 1 - 1e-9, draft.shape)))
    drafted = i32((draft if t == 0 else draft / t + noise).argmax(1))
    if point:
        draft = None
        drafted = i32(target.argmax(1))  # or few would stand
        drafted[::3] = r.integers(0, V, len(drafted[::3]))
    want, acc, near = P.verify(target, draft, starts, drafted, u, t)
    for extra in (dict(), dict(R=len(target) + 3, ld=V + 5, slack=1)):
        tokens, accepted = run(gpu, target, draft, starts, drafted, u, t, **extra)
        assert (tokens[len(want):] == -2).all()
        if near > NEAR:
            assert np.array_equal(tokens[:len(want)], want) and np.array_equal(accepted, acc)
        else:
            assert P.agrees(tokens, accepted, target, draft, starts, drafted, u, t, NEAR)


@pytest.mark.parametrize("point", [False, True])
def test_drawn_tokens_over_the_whole_range_of_the_random_number(gpu, point):
    """one row, many u: every border of the running sum is met from both sides"""
    r = np.random.default_rng(3)
    V, n = 37, 400
    one, other = f32(r.standard_normal((1, V)) * 2), f32(r.standard_normal((1, V)) * 2)
    one[0, [0, 5, 36]] = -np.inf
    target, draft = np.repeat(one, 2 * n, 0), None if point else np.repeat(other, 2 * n, 0)
    drafted = i32(np.full(2 * n, int(other.argmax())))
    u = f32(np.stack([np.full(n, 0.999999), (np.arange(n) + 0.5) / n], 1).ravel())
    u[-1], u[1] = 1.0, 0.0
    starts = i32(2 * np.arange(n + 1))
    want, acc, near = P.verify(target, draft, starts, drafted, u, 1.0)
    got, accepted = run(gpu, target, draft, starts, drafted, u, 1.0)
    assert (acc == 0).all() and np.array_equal(accepted, acc)
    same = got == want
    # u = 0 and u = 1 lie on borders by their nature: the first and the last place with a weight; the others are far from one or compared alone
    for s in range(1, n - 1):
        if not same[2 * s]:
            assert P.verify(target[:2], None if point else draft[:2], [0, 2], drafted[:2], u[2 * s:2 * s + 2], 1.0)[2] < NEAR
    assert same[0] and same[-2] and same.mean() > 0.99


def test_rows_without_a_distribution_and_tokens_that_do_not_exist(gpu):
    r = np.random.default_rng(4)
    V = 300
    target, draft, starts, u = inputs(r, [3] * 9, V)
    drafted = i32(target.argmax(1))
    u[:] = 0.25
    draft[:] = target  # everything stands
    target[3, 17], target[6] = np.nan, -np.inf
    target[9, 4], draft[12, 5] = np.inf, np.nan
    drafted[15], drafted[18] = -1, V
    target[23, 0] = np.nan                             # the row that is drawn from
    target[24:27, 100:], draft[24:27, 100:] = -np.inf, -np.inf
    drafted[24] = int(target[24].argmax())
    for t in (1.0, 0.0):
        want, acc, near = P.verify(target, draft, starts, drafted, u, t)
        got, accepted = run(gpu, target, draft, starts, drafted, u, t)
        assert np.array_equal(got, want) and np.array_equal(accepted, acc)
        assert want[3] == -1 and want[6] == -1 and want[23] == -1 and acc[5] == 0
        assert t == 0 or (want[9] == -1 and want[12] == -1)


def test_equal_maxima_and_equal_distributions(gpu):
    V = 10000
    target = np.zeros((4, V), np.float32)
    target[0, [77, 9000]], target[1, 3] = 5, -1
    got, acc = run(gpu, target, None, [0, 4], [77, 0, 1, 0], np.zeros(4, np.float32), 0.0)
    assert list(got) == [77, 0, 0, -1] and acc[0] == 2
    # p = q: u < 1 stands always; u = 1 never, and what is left of p - q is nothing: drawn from p
    got, acc = run(gpu, target, target, [0, 2, 4], [77, 0, 5, 0], np.array([0.999, 0.5, 1.0, 0.25], np.float32), 1.0)
    want, acc2, _ = P.verify(target, target, [0, 2, 4], [77, 0, 5, 0], np.array([0.999, 0.5, 1.0, 0.25], np.float32), 1.0)
    assert list(acc) == [1, 0] == list(acc2) and got[0] == 77 and list(got[2:]) == [V // 4, -1]
    assert abs(int(got[1]) - int(want[1])) <= 1  # u = 0.5 of an even distribution: the border itself


def test_captured_and_replayed(gpu):
    lib, r = gpu.cuda_lib(), np.random.default_rng(6)
    V, R, n = 5000, 24, 4
    dt, dd, du = zeros(gpu, R * V * 4), zeros(gpu, R * V * 4), zeros(gpu, R * 4)
    ds, dk, tokens, accepted = zeros(gpu, 4 * (n + 1)), zeros(gpu, 4 * R), zeros(gpu, 4 * R), zeros(gpu, 4 * n)
    nbytes = int(lib.ggb_draft_verify_scratch_bytes(R, n))
    scratch = zeros(gpu, nbytes)

    def call():
        gpu.check(lib.ggb_op_draft_verify(dt.ptr, V, dd.ptr, V, V, R, n, ds.ptr, dk.ptr, du.ptr, 1.0, tokens.ptr, accepted.ptr, scratch.ptr, nbytes), "draft_verify")
    graphs = []
    for _ in range(2):  # two graphs on one workspace
        g = C.c_void_p()
        gpu.check(lib.ggb_capture_begin(), "capture")
        call()
        gpu.check(lib.ggb_capture_end(C.byref(g)), "capture")
        graphs.append(g)
    for i, rows in enumerate(([6, 6, 6, 6], [1, 0, 9, 2], [24, 0, 0, 0], [1, 1, 1, 1])):
        target, draft, starts, u = inputs(r, rows, V)
        drafted = i32(draft.argmax(1))
        for b, a in ((dt, target), (dd, draft), (du, u), (ds, starts), (dk, drafted)):
            b.upload(a)
        gpu.check(lib.ggb_graph_launch(graphs[i % 2]), "launch")
        gpu.sync()
        want, acc, near = P.verify(target, draft, starts, drafted, u, 1.0)
        got, accs = tokens.download(np.int32)[:sum(rows)], accepted.download(np.int32)
        assert P.agrees(got, accs, target, draft, starts, drafted, u, 1.0, NEAR) and (near <= NEAR or (np.array_equal(got, want) and np.array_equal(accs, acc)))
    for g in graphs:
        gpu.check(lib.ggb_graph_free(g), "free")


def test_what_is_refused(gpu):
    lib, b = gpu.cuda_lib(), zeros(gpu, 1 << 16)
    p = b.ptr.value
    need = int(lib.ggb_draft_verify_scratch_bytes(2, 1))
    ok = dict(target=p, ld_t=8, draft=p, ld_d=8, V=8, R=2, n_seq=1, starts=p, drafted=p, u=p, t=1.0, tokens=p, accepted=p, scratch=p, nbytes=need)
    for bad in (dict(target=None), dict(starts=None), dict(drafted=None), dict(u=None), dict(tokens=None), dict(accepted=None), dict(scratch=None), dict(V=0), dict(V=1 << 31), dict(R=0),
                dict(R=1 << 16), dict(n_seq=0), dict(n_seq=1 << 16), dict(ld_t=7), dict(ld_d=7), dict(t=-1.0), dict(t=float("nan")), dict(t=float("inf")), dict(t=1e-40),
                dict(nbytes=need - 1), dict(scratch=p + 8)):
        assert lib.ggb_op_draft_verify(*{**ok, **bad}.values()) == -2, bad
        assert b"draft_verify" in lib.ggb_last_error()


@pytest.mark.parametrize("V", [524288 + 32, 600001])
@pytest.mark.parametrize("t", [1.0, 0.0])
def test_vocabularies_of_more_than_64_pieces(gpu, V, t):
    r = np.random.default_rng(30)
    target, draft, starts, u = inputs(r, [3, 1], V)
    drafted = i32(target.argmax(1))
    want, acc, near = P.verify(target, draft, starts, drafted, u, t)
    got, accepted = run(gpu, target, draft, starts, drafted, u, t, ld=V + 3)
    assert np.array_equal(got, want) and np.array_equal(accepted, acc) if near > NEAR else P.agrees(got, accepted, target, draft, starts, drafted, u, t, NEAR)


def test_a_long_row_where_nothing_is_left_of_the_difference(gpu):
    """p = q over 40,000 tokens, u = 1: drawn from p, whose even weights add up exactly"""
    V = 40000
    target = np.zeros((4, V), np.float32)
    got, acc = run(gpu, target, target, [0, 2, 4], [5, 0, 5, 0], np.array([1.0, 0.9, 1.0, 0.125], np.float32), 1.0)
    assert list(acc) == [0, 0] and list(got) == [int(np.floor(np.float64(np.float32(0.9)) * V)), -1, V // 8, -1]


def test_greedy_without_random_numbers(gpu):
    """at temperature 0 neither the draft's logits nor random numbers are read: there need not be any"""
    lib, r = gpu.cuda_lib(), np.random.default_rng(40)
    target, _, starts, _ = inputs(r, [4, 1, 3], 500)
    drafted = i32(target.argmax(1))
    drafted[5] += 1
    nbytes = int(lib.ggb_draft_verify_scratch_bytes(8, 3))
    tokens, accepted, scratch = dev(gpu, np.full(8, -2, np.int32)), dev(gpu, np.full(3, -2, np.int32)), zeros(gpu, nbytes)
    a = [dev(gpu, x) for x in (target, starts, drafted)]
    gpu.check(lib.ggb_op_draft_verify(a[0].ptr, 500, None, 0, 500, 8, 3, a[1].ptr, a[2].ptr, None, 0.0, tokens.ptr, accepted.ptr, scratch.ptr, nbytes), "draft_verify")
    want, acc, _ = P.verify(target, None, starts, drafted, np.zeros(8, np.float32), 0.0)
    assert np.array_equal(tokens.download(np.int32), want) and np.array_equal(accepted.download(np.int32), acc) and list(acc) == [3, 0, 0]


@pytest.mark.parametrize("apart", [0.3, 3e-3, 3e-5])
@pytest.mark.parametrize("V", [300, 50000])
def test_drawn_from_what_little_is_left(gpu, apart, V):
    """drafts that are nearly the target: p - q adds up to some 0.4 apart.  Where one falls, the token that is drawn has a part of the running sum of max(p - q, 0) that u lies in, within the
    bound over that sum: p and q off by NEAR of themselves, so the running sum by 2 NEAR, and u times the whole by that again"""
    r = np.random.default_rng(41)
    n = 60
    target = f32(r.standard_normal((2 * n, V)) * 2.0)
    draft = f32(target + apart * r.standard_normal((2 * n, V)))
    p, q = (np.exp(x.astype(np.float64) - x.max(1, keepdims=True)) for x in (target, draft))
    p, q = p / p.sum(1, keepdims=True), q / q.sum(1, keepdims=True)
    drafted = i32((q - p).argmax(1))  # q above p: u = 1 lets it fall
    u = f32(np.stack([np.ones(n), (np.arange(n) + 0.5) / n], 1).ravel())
    starts = i32(2 * np.arange(n + 1))
    got, accepted = run(gpu, target, draft, starts, drafted, u, 1.0)
    sure = (q > p * (1 + 4 * NEAR))[2 * np.arange(n), drafted[::2]]
    assert sure.sum() > n // 2 and (accepted[sure] == 0).all()
    assert P.agrees(got, accepted, target, draft, starts, drafted, u, 1.0, NEAR)
    for s in np.nonzero(accepted == 0)[0]:
        run_ = np.cumsum(np.maximum(p[2 * s] - q[2 * s], 0))
        v, left, slack = int(got[2 * s]), run_[-1], 4 * NEAR / run_[-1]
        assert run_[v] / left > u[2 * s + 1] - slack and (v == 0 or run_[v - 1] / left <= u[2 * s + 1] + slack)
        assert p[2 * s, v] - q[2 * s, v] > -NEAR * (p[2 * s, v] + q[2 * s, v])  # of the tokens that are left, but for what p and q are off
