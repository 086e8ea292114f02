"""The plain forms of the 8-bit cache and of checked drafts, and what the library says without a device."""
import numpy as np
import pytest

import gemma_ggml_b200 as G
import kv8_plain as P


def test_every_code_comes_back():
    for code in (P.INT8, P.E4M3):
        c = np.arange(256, dtype=np.uint8)
        c = c[c != 128] if code == P.INT8 else c[c & 127 != 127]
        assert np.array_equal(P.encode(code, P.decode(code, c)), c)


def test_rounding_to_the_nearest_code():
    r = np.random.default_rng(0)
    y = np.concatenate([r.uniform(-460, 460, 4000), r.uniform(-0.05, 0.05, 4000)]).astype(np.float32)
    got = P.decode(P.E4M3, P.encode(P.E4M3, y)).astype(np.float64)
    values = np.sort(P.E4M3_VALUES[~np.isnan(P.E4M3_VALUES)])
    want = np.abs(np.clip(y, -448, 448).astype(np.float64)[:, None] - values).min(1)
    assert np.array_equal(np.abs(got - np.clip(y, -448, 448)), want)
    # ties go to the even code: 17 lies between 16 (code 88) and 18 (89), 19 between 18 and 20 (90)
    assert list(P.encode(P.E4M3, np.array([17, 19, -17, 2.0 ** -10, 3 * 2.0 ** -10], np.float32))) == [88, 90, 216, 0, 2]


@pytest.mark.parametrize("code", [P.INT8, P.E4M3])
def test_a_group_filled_token_by_token_is_within_a_step(code):
    r = np.random.default_rng(1)
    x = (r.standard_normal((16, 1, 16)) * np.exp(r.standard_normal((16, 1, 1)))).astype(np.float32)
    c = P.Cache(code, 1, 16, 16, 16, 1)
    for t in range(16):
        P.store(c, x[t:t + 1], x[t:t + 1], x[t:t + 1], [0, 1], [t], [[0]], 0, 0, None, 1.0)
    k, v = c.numbers([0], 16)
    assert np.array_equal(k, v)
    step = c.scales[0, 0, 0, 0] * (1 if code == P.INT8 else np.maximum(2.0 ** -9, 2.0 ** -3 * np.abs(x[:, 0] / c.scales[0, 0, 0, 0])))
    assert (np.abs(k[:, 0] - x[:, 0]) <= step * 1.000001).all()


def test_sizes_of_a_page():
    lib = G.cuda_lib()
    for g, d, dv, b in [(4, 128, 128, 64), (1, 16, 16, 16), (3, 96, 64, 48), (2, 256, 80, 112)]:
        assert lib.ggb_kv8_page_bytes(g, d, dv, b) == P.Cache(P.INT8, g, d, dv, b, 1).pool.size
    for bad in [(0, 64, 64, 64), (1, 24, 64, 64), (1, 64, 272, 64), (1, 64, 64, 40), (1, 64, 0, 64), (1, 64, 64, 0), (1, 64, 64, -16)]:
        assert lib.ggb_kv8_page_bytes(*bad) == 0
    assert G.KV8_INT8 == P.INT8 and G.KV8_E4M3 == P.E4M3


def test_nothing_runs_without_a_device():
    try:
        import torch
        if torch.cuda.is_available():
            pytest.skip("a GPU is present")
    except ImportError:
        pass
    lib, no = G.cuda_lib(), None
    assert lib.ggb_op_kv8_store(1, no, no, no, 1, 1, 1, no, no, 1, 1, 16, 16, 0, 0, no, 1.0, no, 1, 16, no, no) == -3
    assert lib.ggb_op_kv8_attn(0, 1, no, no, no, 1, 16, 1, 1, 1, no, no, 1, 1, 16, 16, 0, 0, 0.0, no, no, 0, no, no, 0) == -3
    assert lib.ggb_op_draft_verify(no, 1, no, 1, 1, 1, 1, no, no, no, 1.0, no, no, no, 0) == -3


def test_drafts_leave_the_targets_distribution():
    """over evenly spread random numbers, the tokens that stand and those drawn in their place together have p's distribution, whatever the draft's"""
    r = np.random.default_rng(2)
    V, n = 5, 40
    target, draft = r.standard_normal((2, V)).astype(np.float32), r.standard_normal((2, V)).astype(np.float32)
    p, q = (np.exp(x - x.max()) / np.exp(x - x.max()).sum() for x in (target[0].astype(np.float64), draft[0].astype(np.float64)))
    got = np.zeros(V)
    for d in range(V):
        for i in range(n):
            for j in range(n):
                tok, _, _ = P.verify(target, draft, [0, 2], [d, 0], np.array([(i + 0.5) / n, (j + 0.5) / n], np.float32), 1.0)
                got[tok[0]] += q[d] / n ** 2
    assert np.abs(got - p).max() < 2.0 / n  # either number is one of n


def test_a_wrong_decision_is_seen():
    r = np.random.default_rng(5)
    V, rows = 2000, [4, 1, 3]
    starts = np.concatenate([[0], np.cumsum(rows)])
    target = r.standard_normal((8, V)).astype(np.float32) * 2
    draft = (target + r.standard_normal((8, V)) * 0.7).astype(np.float32)
    u, drafted = r.random(8).astype(np.float32), draft.argmax(1)
    for d in (draft, None):
        tok, acc, near = P.verify(target, d, starts, drafted, u, 1.0)
        assert P.agrees(tok, acc, target, d, starts, drafted, u, 1.0, 4e-6)
        for s in range(3):
            at = starts[s] + acc[s]
            for other in (tok[at] - 1, tok[at] + 1, -1):
                bad = tok.copy()
                bad[at] = other
                assert other == -1 or abs(other - tok[at]) == 1
                assert not P.agrees(bad, acc, target, d, starts, drafted, u, 1.0, min(4e-6, near / 5))
            bad = acc.copy()
            bad[s] += 1 if acc[s] < rows[s] - 1 else -1
            assert not P.agrees(tok, bad, target, d, starts, drafted, u, 1.0, 4e-6)
