"""Calls at the edges of what the 8-bit paged cache takes: windows and kept positions beyond every length, more sequences than a CTA has threads, a pool off the lines of
128 bytes, infinite queries, two different batches in one captured graph over one workspace.  Plain form and bounds are those of tests/test_kv8_gpu.py."""
import ctypes as C
import types

import numpy as np
import pytest

import kv8_plain as P
from device_util import BF16, F32, at, dev, f32, from_dt, i32, release, zeros
from test_kv8_gpu import batch, check_attention, poison, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _release_buffers():
    yield
    release()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("window,keep", [(1 << 62, 0), (1, 1 << 62), (1 << 40, 1 << 40), (7, 200)])
@pytest.mark.parametrize("new", [[1, 3], [70, 2]])
def test_windows_and_kept_positions_beyond_every_length(gpu, dt, window, keep, new):
    r = np.random.default_rng(11)
    pos = [150, 33]
    starts, tables, pages = batch(r, new, pos, 32)
    cache = P.Cache(P.INT8, 2, 64, 64, 32, pages).filled(r)
    poison(cache, tables, pos, new, True)
    q = f32(r.standard_normal((sum(new), 4, 64)) * 0.2)
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0), min(window, 1 << 30), min(keep, 1 << 30))
    check_attention(dt, run_attention(gpu, dt, cache, q, len(q), starts, pos, tables, max(new), window, keep), want, reach, 64, 220)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("code", [P.INT8, P.E4M3])
def test_more_sequences_than_threads(gpu, dt, code):
    r = np.random.default_rng(12)
    new = [int(x) for x in r.integers(0, 4, 700)]
    new[5], new[699] = 40, 17  # and two for the kernel of portions
    pos = [int(x) for x in r.integers(0, 50, 700)]
    starts, tables, pages = batch(r, new, pos, 16)
    cache = P.Cache(code, 2, 32, 48, 16, pages).filled(r)
    poison(cache, tables, pos, new, True)
    q = f32(r.standard_normal((sum(new), 4, 32)) * 0.3)
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0))
    for scratch in (True, False):
        check_attention(dt, run_attention(gpu, dt, cache, q, len(q) + 1, starts, pos, tables, 40, scratch=scratch), want, reach, 32, 100)


@pytest.mark.parametrize("new", [[2, 1], [90, 1]])
def test_a_pool_off_its_lines(gpu, new):
    """16 bytes behind a boundary of 128: what is asked for of a pool"""
    r = np.random.default_rng(13)
    pos = [100, 65]
    starts, tables, pages = batch(r, new, pos, 64)
    cache = P.Cache(P.E4M3, 2, 128, 96, 64, pages).filled(r)
    q = f32(r.standard_normal((sum(new), 8, 128)) * 0.15)
    raw = dev(gpu, np.concatenate([np.zeros(16, np.uint8), cache.pool.ravel()]))
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0))
    got = run_attention(gpu, F32, cache, q, len(q), starts, pos, tables, max(new), pool=types.SimpleNamespace(ptr=at(raw, 16)))
    check_attention(F32, got, want, reach, 128, 200)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("T", [1, 64])
def test_an_infinite_query_spoils_its_own_row_only(gpu, dt, T):
    r = np.random.default_rng(14)
    starts, tables, pages = batch(r, [T, 2], [100, 30], 64)
    cache = P.Cache(P.INT8, 1, 64, 64, 64, pages).filled(r)
    q = f32(r.standard_normal((T + 2, 2, 64)) * 0.2)
    want, reach = P.attention(cache, q, starts, [100, 30], tables)
    q[0, 0, 5], q[T, 1, 9] = np.inf, -np.inf
    got = run_attention(gpu, dt, cache, q, T + 2, starts, [100, 30], tables, T)
    for t, h in ((0, 0), (T, 1)):
        assert np.isnan(got[t, h]).all()
        got[t, h], want[t, h] = 0, 0
    check_attention(dt, got, want, reach, 64, 200)


def test_two_batches_in_one_graph_over_one_workspace(gpu):
    """steps of one batch and a portion of another behind each other; starts, positions and tables change between replays"""
    lib, r = gpu.cuda_lib(), np.random.default_rng(15)
    H, G, D, B, pages = 8, 2, 64, 32, 40
    cache = P.Cache(P.INT8, G, D, D, B, pages).filled(r)
    pool, nbytes = dev(gpu, cache.pool), int(lib.ggb_kv8_attn_scratch_bytes(D))
    scratch = zeros(gpu, nbytes)
    sides = []
    for T, n in ((6, 4), (90, 2)):
        sides.append(dict(T=T, n=n, q=zeros(gpu, T * H * D * 4), out=zeros(gpu, T * H * D * 4), starts=zeros(gpu, 4 * (n + 1)), pos=zeros(gpu, 4 * n), tables=zeros(gpu, 4 * n * 8)))

    def calls():
        for s in sides:
            gpu.check(lib.ggb_op_kv8_attn(F32, P.INT8, s["q"].ptr, pool.ptr, s["tables"].ptr, 8, B, s["T"], s["T"], s["n"], s["starts"].ptr, s["pos"].ptr, H, G, D, D, 0, 0, 0.0, None, None, 0,
                                          s["out"].ptr, scratch.ptr, nbytes), "kv8_attn")

    def up(buf, a):
        a = np.ascontiguousarray(a)
        gpu.check(lib.ggb_upload(buf.ptr, a.ctypes.data_as(C.c_void_p), a.nbytes), "upload")
        gpu.sync()
    calls()
    gpu.sync()
    gpu.check(lib.ggb_capture_begin(), "capture")
    calls()
    graph = C.c_void_p()
    gpu.check(lib.ggb_capture_end(C.byref(graph)), "capture")
    for news, poss in ((([1, 2, 0, 3], [70, 3, 9, 200]), ([80, 10], [100, 0])), (([1, 1, 1, 1], [0, 31, 32, 140]), ([3, 33], [63, 50]))):
        wants = []
        for s, (new, pos) in zip(sides, (news, poss)):
            tables = i32(r.integers(0, pages, (s["n"], 8)))
            starts, q = i32(np.concatenate([[0], np.cumsum(new)])), f32(r.standard_normal((s["T"], H, D)) * 0.2)
            for name, a in (("q", q), ("starts", starts), ("pos", i32(pos)), ("tables", tables)):
                up(s[name], a)
            wants.append(P.attention(cache, q[:starts[-1]], starts, pos, tables))
        gpu.check(lib.ggb_graph_launch(graph), "graph")
        gpu.sync()
        for s, (want, reach) in zip(sides, wants):
            check_attention(F32, from_dt(F32, s["out"], (s["T"], H, D))[:len(want)], want, reach, D, 256)
    lib.ggb_graph_free(graph)


@pytest.mark.parametrize("new", [1, 40])
def test_fp32_results_over_many_positions(gpu, new):
    """without a workspace a CTA goes through all positions: sums that the tensor cores cut short (by 2^-25 of themselves on average, towards zero, at every step of 16 keys and
    both parts) may not be the long ones.  64 such steps in a row are 1.9e-6 at most, scores and weights add 30 u = 1.8e-6 (all one way; in fact less): 12,000 positions
    in one row would be 1500 / 2 steps"""
    r = np.random.default_rng(16)
    starts, tables, pages = batch(r, [new], [12000], 64)
    cache = P.Cache(P.INT8, 1, 64, 64, 64, pages).filled(r)
    q = f32(r.standard_normal((new, 4, 64)) * 0.2)
    want, _ = P.attention(cache, q, starts, [12000], np.maximum(tables, 0))
    got = run_attention(gpu, F32, cache, q, new, starts, [12000], tables, new, scratch=False)
    assert np.linalg.norm(got - want) < 3.7e-6 * np.linalg.norm(want)
    got = run_attention(gpu, F32, cache, q, new, starts, [12000], tables, new)
    assert np.linalg.norm(got - want) < 3.7e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("H", [33, 64, 128, 129, 256])
def test_many_query_heads_of_one_key_head(gpu, dt, H):
    r = np.random.default_rng(17)
    new, pos = [1, 2, 0, 3], [90, 17, 4, 200]
    starts, tables, pages = batch(r, new, pos, 48)
    cache = P.Cache(P.E4M3, 1, 64, 80, 48, pages).filled(r)
    poison(cache, tables, pos, new, True)
    q = f32(r.standard_normal((6, H, 64)) * 0.2)
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0), 60, 3)
    for scratch in (True, False):
        check_attention(dt, run_attention(gpu, dt, cache, q, 8, starts, pos, tables, 3, 60, 3, scratch=scratch), want, reach, 64, 210)


def test_the_first_call_of_a_process_may_be_captured(tmp_path):
    """what a kernel asks of the driver once is asked for inside a capture"""
    import subprocess
    import sys
    code = """
import ctypes as C, sys
sys.path[:0] = ["tests", "."]
import numpy as np, gemma_ggml_b200 as G, kv8_plain as P
from device_util import F32, dev, f32, from_dt, i32, zeros
G.init()
lib, r = G.cuda_lib(), np.random.default_rng(1)
cache = P.Cache(P.INT8, 1, 64, 64, 64, 4).filled(r)
q, n = f32(r.standard_normal((200, 2, 64)) * 0.2), int(lib.ggb_kv8_attn_scratch_bytes(64))
b = [dev(G, q), dev(G, cache.pool), dev(G, i32([0, 1, 2, 3])), dev(G, i32([0, 200])), dev(G, i32([30])), zeros(G, 200 * 2 * 64 * 4), zeros(G, n)]
G.sync()
G.check(lib.ggb_capture_begin(), "capture")
G.check(lib.ggb_op_kv8_attn(F32, P.INT8, b[0].ptr, b[1].ptr, b[2].ptr, 4, 64, 200, 200, 1, b[3].ptr, b[4].ptr, 2, 1, 64, 64, 0, 0, 0.0, None, None, 0, b[5].ptr, b[6].ptr, n), "kv8_attn")
g = C.c_void_p()
G.check(lib.ggb_capture_end(C.byref(g)), "capture")
G.check(lib.ggb_graph_launch(g), "graph")
G.sync()
want, _ = P.attention(cache, q, [0, 200], [30], i32([[0, 1, 2, 3]]))
got = from_dt(F32, b[5], (200, 2, 64))
assert np.linalg.norm(got - want) < 5e-6 * np.linalg.norm(want)
lib.ggb_graph_free(g)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("new,Dv", [([129], 128), ([143, 161], 112), ([190, 130], 48)])
def test_portions_whose_last_rows_end_inside_a_warp(gpu, dt, new, Dv):
    """rows that end ahead of a warp's others, which go on alone through the output's columns, and rows that see nothing of a tile that others see"""
    r = np.random.default_rng(18)
    pos = [5, 40][:len(new)]
    starts, tables, pages = batch(r, new, pos, 32)
    cache = P.Cache(P.INT8, 1, 64, Dv, 32, pages).filled(r)
    poison(cache, tables, pos, new, True)
    n = int(starts[-1])
    q, gate = f32(r.standard_normal((n, 1, 64)) * 0.2), f32(r.standard_normal((n, 1, Dv)))
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0), 33, 2, gate=gate)
    for scratch in (True, False):
        check_attention(dt, run_attention(gpu, dt, cache, q, n, starts, pos, tables, max(new), 33, 2, gate=gate, scratch=scratch), want, reach, 64, 240)


@pytest.mark.parametrize("dt,D", [(F32, 64), (BF16, 64), (BF16, 256)])
def test_a_ragged_batch_with_room_for_long_sequences(gpu, dt, D):
    """512 sequences whose buffers hold 4,096 tokens, any of them in one sequence, and whose page tables hold a million positions: every sequence with as many items as the longest could have would be
    more than a launch counts, the items that 4,096 tokens can make are not"""
    r = np.random.default_rng(19)
    new = [int(x) for x in r.integers(0, 3, 512)]
    new[100], new[511], new[200:210] = 50, 21, [0] * 10
    pos = [int(x) for x in r.integers(0, 40, 512)]
    starts, few, pages = batch(r, new, pos, 128)
    cache = P.Cache(P.E4M3, 2, D, D, 128, pages).filled(r)
    poison(cache, few, pos, new, True)
    tables = np.full((512, 8192), -1, np.int32)
    tables[:, :few.shape[1]] = few
    q = f32(r.standard_normal((sum(new), 16, D)) * 0.2)
    want, reach = P.attention(cache, q, starts, pos, np.maximum(few, 0))
    for scratch in (True, False):
        got = run_attention(gpu, dt, cache, q, 4096, starts, pos, tables, 4096, scratch=scratch)
        check_attention(dt, got, want, reach, D, 100)
        if scratch:
            assert np.array_equal(got, run_attention(gpu, dt, cache, q, 4096, starts, pos, few, 50))  # the same items in the same order, however they are listed


@pytest.mark.parametrize("dt", [F32, BF16])
def test_one_portion_among_many_steps(gpu, dt):
    """places by tokens: sequences without any, with one and with many rows behind one another"""
    r = np.random.default_rng(20)
    new = [0, 0, 130, 1, 0, 1, 1, 0] + [1] * 90 + [0, 0]
    pos = [int(x) for x in r.integers(0, 300, len(new))]
    starts, tables, pages = batch(r, new, pos, 16)
    cache = P.Cache(P.INT8, 1, 64, 64, 16, pages).filled(r)
    poison(cache, tables, pos, new, True)
    q = f32(r.standard_normal((sum(new), 3, 64)) * 0.2)
    want, reach = P.attention(cache, q, starts, pos, np.maximum(tables, 0), 100, 5)
    for scratch in (True, False):
        check_attention(dt, run_attention(gpu, dt, cache, q, len(q) + 5, starts, pos, tables, 130, 100, 5, scratch=scratch), want, reach, 64, 300)
