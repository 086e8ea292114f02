"""The 8-bit paged cache and checked drafts in plain numpy: what the operators of kv8_store.cu, kv8_attention.cu and draft_verify.cu are compared with.
Storing follows the operators' formulas in 32 bits, number by number (codes and scales are compared bit by bit); attention and probabilities are in 64."""
import numpy as np

GROUP = 16
INT8, E4M3 = 1, 2
TOP = {INT8: 127.0, E4M3: 448.0}
F = np.float32


def e4m3_table():
    """the numbers of the 256 codes: sign, 4 bits of exponent (bias 7), 3 of fraction; no infinities, the last code of either sign is no number"""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if c & 127 == 127 else (-x if c & 128 else x)
    return v


E4M3_VALUES = e4m3_table()


def decode(code, c):
    """uint8 codes -> the whole numbers or 8-bit floating point numbers that they are, float32"""
    return c.view(np.int8).astype(F) if code == INT8 else E4M3_VALUES[c].astype(F)


def encode(code, y):
    """float32 -> the nearest code, ties to the even one, beyond the largest the largest"""
    y = np.clip(y, F(-TOP[code]), F(TOP[code]))
    if code == INT8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    mid = (E4M3_VALUES[:126] + E4M3_VALUES[1:127]) / 2
    a = np.abs(y).astype(np.float64)
    c = np.searchsorted(mid, a, side="left")  # at a middle: the lower code
    tie = (c < 126) & (a == mid[np.minimum(c, 125)]) & (c % 2 == 1)
    c = c + tie
    return (c | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


class Cache:
    """a pool of pages in the operators' layout, as bytes"""

    def __init__(self, code, G, D, Dv, B, pages):
        self.code, self.G, self.D, self.Dv, self.B = code, G, D, Dv, B
        self.record = (B * (D + Dv) + 2 * (B // GROUP) * 4 + 127) // 128 * 128
        self.pool = np.zeros((pages, G, self.record), np.uint8)
        self.k = self.pool[:, :, :B * D].reshape(pages, G, B, D)
        self.v = self.pool[:, :, B * D:B * (D + Dv)].reshape(pages, G, B, Dv)
        at = B * (D + Dv)
        self.scales = self.pool[:, :, at:at + 2 * (B // GROUP) * 4].view(F).reshape(pages, G, 2, B // GROUP)
        for a in (self.k, self.v, self.scales):
            assert np.shares_memory(a, self.pool)

    def filled(self, r, spread=0.4):
        """every page as if tokens had been stored in whole groups"""
        for i, part in enumerate((self.k, self.v)):
            x = (r.standard_normal(part.shape) * np.exp(spread * r.standard_normal((1, self.G, 1, part.shape[3])))).astype(F)
            g = np.abs(x).reshape(*x.shape[:2], self.B // GROUP, -1).max(3) * F(1.0 / TOP[self.code])
            self.scales[:, :, i] = g
            part[...] = encode(self.code, x * (F(1.0) / np.repeat(g, GROUP, 2)[..., None]))
        return self

    def numbers(self, table, n):
        """keys and values of the first n positions, float64 [n][G][D], [n][G][Dv]"""
        j = np.arange(n)
        page, row = np.asarray(table)[j // self.B], j % self.B
        s = self.scales[page, :, :, row // GROUP].astype(np.float64)
        return (decode(self.code, self.k[page, :, row]).astype(np.float64) * s[:, :, 0, None], decode(self.code, self.v[page, :, row]).astype(np.float64) * s[:, :, 1, None])


def turned(x, cs, rot, halves):
    """x float32 [..., D], cs [rot / 2][cos, sin]"""
    y = x.copy()
    if rot:
        h = rot // 2
        a, b = (x[..., :h], x[..., h:rot]) if halves else (x[..., 0:rot:2], x[..., 1:rot:2])
        first, second = a * cs[:, 0] - b * cs[:, 1], a * cs[:, 1] + b * cs[:, 0]
        if halves:
            y[..., :h], y[..., h:rot] = first, second
        else:
            y[..., 0:rot:2], y[..., 1:rot:2] = first, second
    return y


def store(cache, q, k, v, starts, pos0, tables, rot, halves, cos_sin, scale):
    """q [T][H][D], k [T][G][D], v [T][G][Dv] float32; writes the cache, returns the turned queries (rows of no sequence: NaN)"""
    q_out = np.full(q.shape, np.nan, F)
    code = cache.code
    for s in range(len(pos0)):
        t0, n, p0 = int(starts[s]), int(starts[s + 1] - starts[s]), int(pos0[s])
        cs = [cos_sin[p0 + i] if rot else None for i in range(n)]
        for i in range(n):
            q_out[t0 + i] = turned(q[t0 + i], cs[i], rot, halves) * F(scale)
        new = [(np.stack([turned(k[t0 + i], cs[i], rot, halves) for i in range(n)]) if n else None, cache.k), (v[t0:t0 + n], cache.v)]
        for grp in range(p0 // GROUP, (p0 + n - 1) // GROUP + 1 if n else p0 // GROUP):
            first = grp * GROUP
            page, row0 = int(tables[s][first // cache.B]), first % cache.B
            held, end = max(0, p0 - first), min(GROUP, p0 + n - first)
            for kind, (x, part) in enumerate(new):
                y = x[first + held - p0:first + end - p0]  # [rows][G][n]
                y = np.where(np.isnan(y), F(0), y)
                mag = np.where(np.isinf(y), F(0), np.abs(y)).max((0, 2))
                least = np.where(mag > 0, np.maximum(mag * F(1.0 / TOP[code]), F(2.0 ** -100)), F(0))
                for g in range(cache.G):
                    old = cache.scales[page, g, kind, row0 // GROUP] if held else F(0)
                    new_scale = max(least[g], F(2) * old) if least[g] > old else old
                    if new_scale > old and held:
                        c = part[page, g, row0:row0 + held]
                        part[page, g, row0:row0 + held] = encode(code, decode(code, c) * (old / new_scale))
                    inv = F(1) / (new_scale if new_scale > 0 else F(1))
                    with np.errstate(invalid="ignore"):
                        part[page, g, row0 + held:row0 + end] = encode(code, y[:, g] * inv)
                    cache.scales[page, g, kind, row0 // GROUP] = new_scale
    return q_out


def attention(cache, q, starts, pos0, tables, window=0, keep=0, cap=0.0, sink=None, gate=None):
    """q [T][H][D] -> float64 [T][H][Dv] (rows of no sequence: NaN), and per row the largest sum of |q_d k_d| and |value| it met"""
    T, H, _ = q.shape
    out, reach = np.full((T, H, cache.Dv), np.nan), np.zeros((T, H, 2))
    for s in range(len(pos0)):
        t0, n, p0 = int(starts[s]), int(starts[s + 1] - starts[s]), int(pos0[s])
        if not n:
            continue
        k, v = cache.numbers(tables[s], p0 + n)
        for i in range(n):
            at = p0 + i
            j = np.arange(at + 1)
            j = j[(at - j < window) | (j < keep)] if window > 0 else j
            for h in range(H):
                g = h // (H // cache.G)
                x = q[t0 + i, h].astype(np.float64)
                z = k[j, g] @ x
                if cap > 0:
                    z = cap * np.tanh(z / cap)
                m = max(z.max(), sink[h]) if sink is not None else z.max()
                w = np.exp(z - m)
                o = w @ v[j, g] / (w.sum() + (np.exp(sink[h] - m) if sink is not None else 0.0))
                out[t0 + i, h] = o / (1 + np.exp(-gate[t0 + i, h].astype(np.float64))) if gate is not None else o
                reach[t0 + i, h] = (np.abs(k[j, g]) @ np.abs(x)).max(), np.abs(v[j, g]).max()
    return out, reach


def verify(target, draft, starts, drafted, u, temperature):
    """tokens (int, -1 behind the drawn one; rows of no sequence -2), accepted, and how near the nearest decision was: of u q against p, relative, and of the running
    sum, in parts of the whole"""
    n = len(starts) - 1
    tokens, accepted, near = np.full(len(target), -2, np.int64), np.zeros(n, np.int64), np.inf

    def soft(x):
        x = x.astype(np.float64)
        if np.isnan(x).any() or np.isposinf(x).any() or not (x > -np.inf).any():
            return None
        e = np.exp((x - x.max()) / temperature)
        return e / e.sum()

    for s in range(n):
        r0, rows = int(starts[s]), int(starts[s + 1] - starts[s])
        if rows == 0:
            continue
        tokens[r0:r0 + rows] = -1
        a = 0
        while True:
            row = target[r0 + a]
            if temperature == 0:
                best = -1 if np.isnan(row).any() or not (row > -np.inf).any() else int(np.argmax(row))
                stands = a < rows - 1 and best >= 0 and drafted[r0 + a] == best
            else:
                p, d = soft(row), int(drafted[r0 + a])
                q = soft(draft[r0 + a]) if draft is not None and a < rows - 1 else None
                stands = False
                if a < rows - 1 and p is not None and (draft is None or q is not None) and 0 <= d < len(p):
                    left = float(u[r0 + a]) * (q[d] if draft is not None else 1.0)
                    stands = left < p[d]
                    near = min(near, abs(left - p[d]) / max(p[d], 1e-300))
            if not stands:
                break
            tokens[r0 + a] = drafted[r0 + a]
            a += 1
        accepted[s] = a
        if temperature == 0:
            tokens[r0 + a] = best
            continue
        if p is None or (a < rows - 1 and draft is not None and q is None):
            continue
        w = p
        if a < rows - 1:
            rest = p.copy()
            if draft is not None:
                rest = np.maximum(p - q, 0)
            elif 0 <= d < len(p):
                rest[d] = 0
            w = rest if rest.sum() > 0 else p
        run = np.cumsum(w)
        at = float(u[r0 + rows - 1]) * run[-1]
        v = int((run <= at).sum())
        v = min(v, int(np.nonzero(w > 0)[0][-1]))
        tokens[r0 + a] = v
        near = min(near, float(np.abs(run - at).min() / run[-1]))
    return tokens, accepted, near


def agrees(tokens, accepted, target, draft, starts, drafted, u, temperature, near):
    """whether every decision behind `tokens` and `accepted` is one that exponentials, each off by up to `near` of itself, can lead to (every row has a distribution):
    follows them, row by row, with p and q in 64 bits"""
    def soft(x):
        e = np.exp((x.astype(np.float64) - float(x.max())) / temperature)
        return e / e.sum()

    for s in range(len(starts) - 1):
        r0, rows = int(starts[s]), int(starts[s + 1] - starts[s])
        if rows == 0:
            if accepted[s] != 0:
                return False
            continue
        a = int(accepted[s])
        if not 0 <= a < rows or (tokens[r0:r0 + a] != drafted[r0:r0 + a]).any() or (tokens[r0 + a + 1:r0 + rows] != -1).any():
            return False
        for j in range(min(a + 1, rows - 1)):
            d, p = int(drafted[r0 + j]), soft(target[r0 + j])
            left = float(u[r0 + j]) * (soft(draft[r0 + j])[d] if draft is not None else 1.0)
            if not (left < p[d] * (1 + 2 * near) if j < a else left > p[d] * (1 - 2 * near)):  # either side is off
                return False
        w, slack, v = soft(target[r0 + a]), near, int(tokens[r0 + a])
        if a < rows - 1 and draft is not None:
            w, slack = np.maximum(w - soft(draft[r0 + a]), 0), 2 * near
        elif a < rows - 1:
            w[int(drafted[r0 + a])] = 0
        run = np.cumsum(w)
        at = float(u[r0 + rows - 1]) * run[-1]
        if not 0 <= v < len(w) or not run[v] > at - 2 * slack or not (v == 0 or run[v - 1] <= at + 2 * slack):  # the running sum and the whole
            return False
    return True
