"""Serving a batch of sequences from an 8-bit paged cache: what the operators are measured on.

Three operators, called one behind the other when a target model checks the tokens that a smaller model has drafted:

  store    ggb_op_kv8_store: new keys and values, turned by their positions, into an 8-bit paged cache with a scale per 16 tokens and head; the
           queries turned beside them
  attn     ggb_op_kv8_attn: grouped-query soft-max attention over that cache, from one token per sequence to whole portions
  verify   ggb_op_draft_verify: which drafted tokens stand against the target's probabilities, by given random numbers, and the token behind them

A case is a plain dict; `kind` picks the operator.  The sequences' lengths follow from the case alone, everything else from the seed.
"""
import math

import torch

own = False

GROUP = 16  # tokens that share a scale
CODES = {"int8": (1, torch.int8, 127.0), "e4m3": (2, torch.float8_e4m3fn, 448.0)}
TYPES = {"bf16": (30, torch.bfloat16), "f32": (0, torch.float32)}


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the smallest calls: one sequence, one token
        dict(name="store_step_1", kind="store", code="int8", seqs=1, new=1, mix=False, pos=777, heads=16, kv=4, dim=128, vdim=128, rot=128, halves=True, page=64),
        dict(name="attn_step_1", kind="attn", dt="bf16", code="int8", seqs=1, new=1, mix=False, pos=777, heads=16, kv=4, dim=128, vdim=128, window=0, keep=0,
             softcap=0.0, sink=False, gate=False, page=64),
        dict(name="verify_1", kind="verify", seqs=1, drafts=4, vocab=32000, temperature=0.8, point=False),
        # a step of a served batch, ragged lengths
        dict(name="store_step_64", kind="store", code="e4m3", seqs=64, new=1, mix=False, pos=4000, heads=32, kv=8, dim=128, vdim=128, rot=64, halves=False, page=64),
        dict(name="attn_step_32", kind="attn", dt="bf16", code="int8", seqs=32, new=1, mix=False, pos=8000, heads=32, kv=8, dim=128, vdim=128, window=0, keep=0,
             softcap=0.0, sink=False, gate=False, page=64),
        # up to four drafted tokens and the one before them, the float32 engine: window, kept first tokens, soft cap, sink
        dict(name="attn_drafts_f32", kind="attn", dt="f32", code="e4m3", seqs=12, new=5, mix=False, pos=3001, heads=12, kv=4, dim=96, vdim=64, window=2000, keep=4,
             softcap=30.0, sink=True, gate=False, page=48),
        # one long sequence, few key heads: its keys are all there is to spread
        dict(name="attn_long_1", kind="attn", dt="bf16", code="e4m3", seqs=1, new=1, mix=False, pos=100001, heads=8, kv=1, dim=256, vdim=256, window=0, keep=0,
             softcap=0.0, sink=False, gate=False, page=128),
        # a prompt's second portion: window, kept first tokens, gate
        dict(name="attn_portion_1024", kind="attn", dt="bf16", code="int8", seqs=1, new=1024, mix=False, pos=1024, heads=16, kv=4, dim=128, vdim=128, window=1024,
             keep=4, softcap=0.0, sink=False, gate=True, page=64),
        # a portion beside sequences that decode, the float32 engine
        dict(name="attn_mixed_f32", kind="attn", dt="f32", code="int8", seqs=9, new=777, mix=True, pos=2000, heads=16, kv=4, dim=128, vdim=128, window=0, keep=0,
             softcap=0.0, sink=False, gate=False, page=64),
        # two prompts at once
        dict(name="store_portion_4096", kind="store", code="int8", seqs=2, new=2731, mix=False, pos=1001, heads=32, kv=8, dim=128, vdim=128, rot=128, halves=True, page=64),
        # Gemma's vocabulary, a batch that samples, and one that is greedy behind drafts without probabilities
        dict(name="verify_16", kind="verify", seqs=16, drafts=5, vocab=256000, temperature=1.0, point=False),
        dict(name="verify_greedy_24", kind="verify", seqs=24, drafts=7, vocab=49999, temperature=0.0, point=True),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        """a multiple of `step` in [lo, hi], even over the logarithm"""
        return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))) / step)) * step)

    kind = rng.choice(["store", "attn", "attn", "attn", "attn", "verify", "verify"])
    if kind == "verify":
        c = dict(kind=kind, seqs=size(1, 32), drafts=rng.randint(0, 8), vocab=size(1000, 256000), temperature=rng.choice([0.0, 0.6, 1.0, 1.3]), point=rng.random() < 0.3)
        while c["seqs"] * (c["drafts"] + 1) * c["vocab"] > 24e6:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["drafts"] = max(0, c["drafts"] - 1)
        return c
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 128, 192, 256])
    c = dict(kind=kind, code=rng.choice(["int8", "e4m3"]), heads=kv * rng.choice([1, 2, 4, 8]), kv=kv, dim=dim, vdim=rng.choice([dim, 64, 128]), page=rng.choice([16, 48, 64, 128]))
    if kind == "store":
        c.update(seqs=size(1, 64), new=rng.choice([1, 1, size(2, 16), size(16, 2048)]), mix=rng.random() < 0.3, pos=rng.choice([0, size(1, 4000)]),
                 rot=rng.choice([0, 32, 64, dim]), halves=rng.random() < 0.5)
        while c["seqs"] * c["new"] * (c["heads"] + c["kv"]) * dim > 18e6:
            c["seqs"], c["new"] = max(1, c["seqs"] // 2), max(1, c["new"] * 3 // 4)
        return c
    c.update(dt=rng.choice(["bf16", "bf16", "f32"]), seqs=size(1, 48), new=rng.choice([1, 1, size(2, 8), size(9, 1024)]), mix=rng.random() < 0.3,
             pos=rng.choice([0, size(1, 9000), size(1, 9000)]), window=rng.choice([0, 0, 128, 1024]), softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.3,
             gate=rng.random() < 0.2)
    c["keep"] = rng.choice([0, 4, 50]) if c["window"] else 0
    # what the plain form holds: the scores of all heads and the cache in 32 bits
    while c["seqs"] * c["heads"] * c["new"] * (c["pos"] + c["new"]) > 3e8 or c["seqs"] * c["kv"] * (dim + c["vdim"]) * (c["pos"] + c["new"]) > 4e8:
        c["seqs"] = c["seqs"] * 2 // 3 if c["seqs"] > 1 else 1
        c["pos"] = c["pos"] * 3 // 4
        c["new"] = max(1, c["new"] * 4 // 5)
    return c


def lengths(c):
    """tokens that each sequence brings, and how many it has in the cache already"""
    n = c["seqs"]
    ragged = [((s * 40503 + 11) % 97) / 96.0 for s in range(n)]
    if c["mix"]:  # the first brings a portion, the others a token each
        new = [c["new"]] + [1] * (n - 1)
    else:
        new = [c["new"] if s == 0 else 1 + int(ragged[s] * (c["new"] - 1)) for s in range(n)]
    pos = [c["pos"] if s == 0 else int(c["pos"] * (0.25 + 0.75 * ragged[n - 1 - s])) for s in range(n)]
    return new, pos


def record_bytes(c):
    """a head's part of a page: codes of the keys, codes of the values, 16 tokens' scales of either, in whole 128 bytes"""
    return (c["page"] * (c["dim"] + c["vdim"]) + 2 * (c["page"] // GROUP) * 4 + 127) // 128 * 128


# ------------------------------------------------------------------------------------------------------------ inputs
class State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def maker(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 12345)
    return g


def views(c, pool):
    """the parts of a pool of pages [pages][kv][record]: codes of keys and values, scales [pages][kv][2][page / 16]"""
    pages, B, D, Dv = pool.shape[0], c["page"], c["dim"], c["vdim"]
    ct = CODES[c["code"]][1]
    k = pool[:, :, :B * D].unflatten(2, (B, D)).view(ct)
    v = pool[:, :, B * D:B * (D + Dv)].unflatten(2, (B, Dv)).view(ct)
    at = B * (D + Dv) // 4
    sc = pool.view(torch.float32)[:, :, at:at + 2 * (B // GROUP)].unflatten(2, (2, B // GROUP))
    return k, v, sc


def encode(x, scale, code):
    """numbers over their scale, rounded into 8 bits"""
    _, ct, top = CODES[code]
    y = (x * (1.0 / torch.where(scale > 0, scale, torch.ones_like(scale)))).clamp(-top, top)
    return y.round().to(ct) if code == "int8" else y.to(ct)


def fill_cache(c, g, pages):
    """a pool whose every page holds tokens: keys and values of ordinary size, coordinates of different strength"""
    B, G, D, Dv = c["page"], c["kv"], c["dim"], c["vdim"]
    pool = torch.zeros(pages, G, record_bytes(c), dtype=torch.uint8, device="cuda")
    k, v, sc = views(c, pool)
    top = CODES[c["code"]][2]
    for i, (part, n) in enumerate(((k, D), (v, Dv))):
        strength = torch.exp(0.3 * torch.randn(G, 1, n, generator=g, device="cuda"))
        step = max(1, (1 << 26) // (G * B * n))
        for p in range(0, pages, step):
            x = torch.randn(min(step, pages - p), G, B, n, generator=g, device="cuda") * strength
            s = x.unflatten(2, (B // GROUP, GROUP)).abs().amax((3, 4)) / top
            sc[p:p + step, :, i] = s
            part[p:p + step].view(torch.uint8).copy_(encode(x, s.repeat_interleave(GROUP, 2)[..., None], c["code"]).view(torch.uint8))
    return pool


def prepare(case, seed):
    c, g = case, maker(seed)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["kind"] == "verify":
        n, V = c["seqs"], c["vocab"]
        rows = [1 + (c["drafts"] if s == 0 else (s * 5 + c["drafts"]) % (c["drafts"] + 1)) for s in range(n)]
        R = sum(rows)
        starts = i32([sum(rows[:s]) for s in range(n + 1)])
        target = torch.randn(R, V, generator=g, device="cuda") * 2.5
        draft = None if c["point"] else target + torch.randn(R, V, generator=g, device="cuda") * 0.7  # a smaller model's: near the target's, not equal
        seen = (target + torch.randn(R, V, generator=g, device="cuda") * 0.05) if c["point"] else draft
        noise = -torch.log(-torch.log(torch.rand(R, V, generator=g, device="cuda").clamp(1e-12, 1 - 1e-7)))
        drafted = (seen if c["temperature"] == 0 else seen / c["temperature"] + noise).argmax(1).to(torch.int32)
        u = torch.rand(R, generator=g, device="cuda")
        st = State(c=c, R=R, rows=rows, starts=starts, target=target, draft=draft, drafted=drafted, u=u, tokens=torch.full((R,), -1, dtype=torch.int32, device="cuda"),
                   accepted=torch.zeros(n, dtype=torch.int32, device="cuda"), scratch=torch.zeros(64 + 16 * (R * 2 * 132 + n * 132), dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        return st
    new, pos = lengths(c)
    n, B, G, D, Dv, H = c["seqs"], c["page"], c["kv"], c["dim"], c["vdim"], c["heads"]
    T = sum(new)
    need = [(p + t + B - 1) // B for p, t in zip(pos, new)]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    wide = max(need) + 1
    table = torch.zeros(n, wide, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(n):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    st = State(c=c, T=T, table=table, wide=wide, starts=i32([sum(new[:s]) for s in range(n + 1)]), pos=i32(pos), most=max(new), reach=max(p + t for p, t in zip(pos, new)),
               pool=fill_cache(c, g, pages))
    if c["kind"] == "store":
        ld = (H + G) * D + G * Dv
        st.x = torch.randn(T, ld, generator=g, device="cuda") * torch.exp(0.3 * torch.randn(1, ld, generator=g, device="cuda"))
        half = c["rot"] // 2
        ang = torch.arange(st.reach, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
        st.cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        st.q = torch.empty(T, H, D, device="cuda")
        st.scale = D ** -0.5
    else:
        st.q = torch.randn(T, H, D, generator=g, device="cuda") * (1.5 * D ** -0.5)
        st.sink = torch.randn(H, generator=g, device="cuda") if c["sink"] else None
        st.gate = torch.randn(T, H, Dv, generator=g, device="cuda") if c["gate"] else None
        st.out = torch.empty(T, H, Dv, dtype=TYPES[c["dt"]][1], device="cuda")
        st.scratch = torch.zeros(scratch_bytes(c), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return st


def scratch_bytes(c):
    """room for the parts of rows whose keys are spread: 512 blocks, twice 32 rows each"""
    return 512 * 2 * 32 * (c["vdim"] + 4) * 4


# ------------------------------------------------------------------------------------------------------------ plain forms
def token_places(s):
    """of every new token: its sequence and its position there"""
    t = torch.arange(s.T, device="cuda")
    seq = torch.searchsorted(s.starts[1:].long(), t, right=True)
    return seq, s.pos.long()[seq] + t - s.starts.long()[seq]


def turned(c, x, cs):
    """the pairs of a head's first `rot` numbers turned by [tokens][rot / 2][cos, sin]"""
    r = c["rot"]
    if r == 0:
        return x
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if c["halves"] else (x[..., 0:r:2], x[..., 1:r:2])
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]
    y = [a * co - b * si, b * co + a * si]
    return torch.cat([torch.cat(y, -1) if c["halves"] else torch.stack(y, -1).flatten(-2), x[..., r:]], -1)


def plain_store(s):
    c = s.c
    H, G, D, Dv, B = c["heads"], c["kv"], c["dim"], c["vdim"], c["page"]
    top = CODES[c["code"]][2]
    seq, p = token_places(s)
    cs = s.cs[p]
    q, k, v = s.x.split([H * D, G * D, G * Dv], 1)
    s.q.copy_(turned(c, q.unflatten(1, (H, D)), cs) * s.scale)
    page, row = s.table.long()[seq, p // B], p % B
    # the group that a sequence's first new token falls into may hold tokens of earlier calls
    first, held = s.pos.long(), s.pos.long() % GROUP
    fpage = s.table.long().gather(1, (first // B)[:, None])[:, 0]
    fgroup = first % B // GROUP
    brings = s.starts[1:] > s.starts[:-1]
    kc, vc, sc = views(c, s.pool)
    for i, (x, part) in enumerate(((turned(c, k.unflatten(1, (G, D)), cs), kc), (v.unflatten(1, (G, Dv)), vc))):
        most = torch.zeros(sc.shape[0] * (B // GROUP), G, device="cuda").index_reduce_(0, page * (B // GROUP) + row // GROUP, x.abs().amax(2), "amax")
        most = most.unflatten(0, (sc.shape[0], B // GROUP)).transpose(1, 2)
        least = torch.where(most > 0, (most * (1.0 / top)).clamp_min(2.0 ** -100), torch.zeros_like(most))
        here = torch.zeros(sc.shape[0], B // GROUP, dtype=torch.bool, device="cuda")
        here[page, row // GROUP] = True
        old = torch.zeros_like(least)
        old[fpage, :, fgroup] = torch.where((brings & (held > 0))[:, None], sc[fpage, :, i, fgroup], 0.0)
        scale = torch.where(least > old, torch.maximum(least, 2.0 * old), old)
        # what stands there already, over its group's larger scale
        before, after = old[fpage, :, fgroup][:, :, None, None], scale[fpage, :, fgroup][:, :, None, None]
        rows = fgroup[:, None] * GROUP + torch.arange(GROUP, device="cuda")
        codes = part[fpage[:, None], :, rows].transpose(1, 2)  # [sequences][kv][16][n]
        again = codes.float() * (before / torch.where(after > 0, after, 1.0))
        again = again.round().to(codes.dtype) if c["code"] == "int8" else again.to(codes.dtype)
        keep = (torch.arange(GROUP, device="cuda") < held[:, None])[:, None, :, None] & (after > before) & brings[:, None, None, None]
        bits = torch.where(keep, again.view(torch.uint8), codes.view(torch.uint8))
        raw = part.view(torch.uint8)
        raw[fpage[:, None], :, rows] = bits.transpose(1, 2)
        raw[page, :, row] = encode(x, scale[page, :, row // GROUP][..., None], c["code"]).view(torch.uint8)
        sc[:, :, i] = torch.where(here[:, None], scale, sc[:, :, i])
    return dict(q=s.q, k=kc, v=vc, scales=sc)


def plain_attn(s):
    c = s.c
    H, G, B, D, Dv, n = c["heads"], c["kv"], c["page"], c["dim"], c["vdim"], c["seqs"]
    kc, vc, sc = views(c, s.pool)
    j = torch.arange(s.reach, device="cuda")
    page, row = s.table.long()[:, j // B], j % B
    k = kc.view(torch.uint8)[page, :, row].view(kc.dtype).float() * sc[page, :, 0, row // GROUP][..., None]  # [sequences][keys][kv][D]
    v = vc.view(torch.uint8)[page, :, row].view(vc.dtype).float() * sc[page, :, 1, row // GROUP][..., None]
    seq, p = token_places(s)
    place = p - s.pos.long()[seq]
    q = torch.zeros(n, s.most, H, D, device="cuda")
    q[seq, place] = s.q
    q = q.unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [sequences][kv][heads of it x tokens][D]
    score = (q @ k.permute(0, 2, 3, 1)).unflatten(2, (H // G, s.most))
    if c["softcap"] > 0:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    i = s.pos.long()[:, None, None] + torch.arange(s.most, device="cuda")[None, :, None]
    seen = j <= i
    if c["window"] > 0:
        seen = seen & ((i - j < c["window"]) | (j < c["keep"]))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    w = torch.exp(score - most)
    total = w.sum(-1, keepdim=True)
    if c["sink"]:
        total = total + torch.exp(s.sink.view(1, G, H // G, 1, 1) - most)
    o = (w / total).flatten(2, 3) @ v.permute(0, 2, 1, 3)
    o = o.unflatten(2, (H // G, s.most)).permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, place]
    if c["gate"]:
        o = o * torch.sigmoid(s.gate)
    return o.to(s.out.dtype)


def plain_verify(s):
    c = s.c
    n, V, K = c["seqs"], c["vocab"], c["drafts"]
    start, rows = s.starts[:-1].long(), (s.starts[1:] - s.starts[:-1]).long()
    at = torch.arange(K + 1, device="cuda")[None].minimum(rows[:, None] - 1) + start[:, None]  # [sequences][rows]; past the end the last one again
    token = s.drafted.long()[at]
    drafts = torch.arange(K + 1, device="cuda")[None] < rows[:, None] - 1
    if c["temperature"] == 0:
        best = s.target.argmax(1)
        good = best[at] == token
    else:
        p = torch.softmax(s.target.double() / c["temperature"], 1)
        q = None if s.draft is None else torch.softmax(s.draft.double() / c["temperature"], 1)
        good = s.u.double()[at] * (1.0 if q is None else q[at, token]) < p[at, token]
    stands = (good & drafts).long().cumprod(1)
    taken = stands.sum(1)
    last = start + taken
    if c["temperature"] == 0:
        extra = best[last]
    else:
        w = p[last]
        rejected = (taken < rows - 1)[:, None]
        if q is None:
            rest = w.scatter(1, s.drafted.long()[last][:, None], 0.0)
        else:
            rest = (w - q[last]).clamp_min(0.0)
        w = torch.where(rejected & (rest.sum(1, keepdim=True) > 0), rest, w)
        run_ = w.cumsum(1)
        extra = (run_ <= s.u.double()[start + rows - 1][:, None] * run_[:, -1:]).sum(1)
        extra = extra.minimum((w > 0).long().cumsum(1).argmax(1))
    s.tokens.fill_(-1)
    s.tokens[at] = torch.where(stands.bool(), token, -1).to(torch.int32)
    s.tokens[last] = extra.to(torch.int32)
    s.accepted.copy_(taken)
    return dict(tokens=s.tokens, accepted=s.accepted)


# ------------------------------------------------------------------------------------------------------------ the calls
LIBRARY = []


def ptr(t, offset=0):
    return t.data_ptr() + offset if t is not None else None


def call(name, *args):
    if not LIBRARY:
        import gemma_ggml_b200 as G
        G.init()
        LIBRARY.extend((G, G.cuda_lib()))
    G, lib = LIBRARY
    G.check(getattr(lib, name)(*args), name)


def run(state):
    s, c = state, state.c
    if not own:
        return {"store": plain_store, "attn": plain_attn, "verify": plain_verify}[c["kind"]](s)
    if c["kind"] == "verify":
        V = c["vocab"]
        call("ggb_op_draft_verify", ptr(s.target), V, ptr(s.draft), V, V, s.R, c["seqs"], ptr(s.starts), ptr(s.drafted), ptr(s.u), c["temperature"], ptr(s.tokens), ptr(s.accepted),
             ptr(s.scratch), s.scratch.numel())
        return dict(tokens=s.tokens, accepted=s.accepted)
    H, G, D, Dv = c["heads"], c["kv"], c["dim"], c["vdim"]
    code = CODES[c["code"]][0]
    if c["kind"] == "store":
        ld = s.x.shape[1]
        call("ggb_op_kv8_store", code, ptr(s.x), ptr(s.x, 4 * H * D), ptr(s.x, 4 * (H + G) * D), ld, s.T, c["seqs"], ptr(s.starts), ptr(s.pos), H, G, D, Dv, c["rot"],
             int(c["halves"]), ptr(s.cs) if c["rot"] else None, s.scale, ptr(s.table), s.wide, c["page"], ptr(s.pool), ptr(s.q))
        k, v, sc = views(c, s.pool)
        return dict(q=s.q, k=k, v=v, scales=sc)
    call("ggb_op_kv8_attn", TYPES[c["dt"]][0], code, ptr(s.q), ptr(s.pool), ptr(s.table), s.wide, c["page"], s.T, s.most, c["seqs"], ptr(s.starts), ptr(s.pos), H, G, D, Dv, c["window"],
         c["keep"], c["softcap"], ptr(s.sink), ptr(s.gate), H * Dv, ptr(s.out), ptr(s.scratch), s.scratch.numel())
    return s.out


# ------------------------------------------------------------------------------------------------------------ work and 64 bits
def work(case):
    c = case
    if c["kind"] == "verify":
        rows = sum(1 + (c["drafts"] if s == 0 else (s * 5 + c["drafts"]) % (c["drafts"] + 1)) for s in range(c["seqs"]))
        sides = 1 if c["point"] else 2
        # the last row of a sequence has no drafted token to judge
        return dict(bytes=4 * c["vocab"] * (rows + (rows - c["seqs"]) * (sides - 1)), flops=3 * c["vocab"] * rows * sides)
    new, pos = lengths(c)
    H, G, D, Dv, T = c["heads"], c["kv"], c["dim"], c["vdim"], sum(new)
    if c["kind"] == "store":
        held = sum(p % GROUP for p in pos)  # codes of earlier tokens that share a group with new ones
        return dict(bytes=4 * T * ((2 * H + G) * D + G * Dv) + T * G * (D + Dv) + held * G * (D + Dv) // 2, flops=T * (3 * (H + G) * D + 3 * G * (D + Dv)))
    size = 2 if c["dt"] == "bf16" else 4
    keys = pairs = 0
    for t, p in zip(new, pos):
        w, keep = c["window"], c["keep"]
        if w <= 0:
            keys += p + t
            pairs += t * p + t * (t + 1) // 2
            continue
        low = max(0, p - w + 1)
        keys += p + t - low + min(keep, low)
        for i in range(p, p + t):
            lo = max(0, i - w + 1)
            pairs += i + 1 - lo + min(keep, lo)
    return dict(bytes=keys * G * (D + Dv) + 2 * 4 * keys * G // GROUP + T * H * (4 * D + size * Dv) + (4 * T * H * Dv if c["gate"] else 0), flops=2 * pairs * H * (D + Dv))


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "verify":
        return None  # whole numbers
    H, G, B, D, Dv = c["heads"], c["kv"], c["page"], c["dim"], c["vdim"]
    new, pos = lengths(c)
    if c["kind"] == "store":
        q = s.x[:, :H * D].double().reshape(s.T, H, D)
        at = torch.cat([torch.arange(p, p + t, device="cuda") for t, p in zip(new, pos)])
        r = c["rot"] // 2
        out = q.clone()
        if r:
            z = torch.complex(s.cs[at, :, 0].double(), s.cs[at, :, 1].double())[:, None]
            pair = torch.complex(q[..., :r], q[..., r:2 * r]) if c["halves"] else torch.view_as_complex(q[..., :2 * r].reshape(s.T, H, r, 2))
            z = pair * z
            if c["halves"]:
                out[..., :r], out[..., r:2 * r] = z.real, z.imag
            else:
                out[..., :2 * r] = torch.view_as_real(z).reshape(s.T, H, 2 * r)
        return dict(q=out * s.scale, k=None, v=None, scales=None)  # the codes are what the rule makes of 32-bit numbers
    kc, vc, sc = views(c, s.pool)
    out = torch.empty(s.T, H, Dv, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (t, p) in enumerate(zip(new, pos)):
        n = p + t
        pages = s.table[b, :(n + B - 1) // B].long()
        step = sc[pages].double().repeat_interleave(GROUP, 3)  # [pages][kv][2][B]
        k = (kc[pages].double() * step[:, :, 0, :, None]).transpose(0, 1).reshape(G, -1, D)[:, :n]
        v = (vc[pages].double() * step[:, :, 1, :, None]).transpose(0, 1).reshape(G, -1, Dv)[:, :n]
        i, j = torch.arange(p, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        hidden = j > i
        if c["window"] > 0:
            hidden |= (j <= i - c["window"]) & (j >= c["keep"])
        for h in range(H):
            z = s.q[t0:t0 + t, h].double() @ k[h // (H // G)].T
            if c["softcap"] > 0:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            z[hidden] = -math.inf
            if c["sink"]:
                z = torch.cat([z, s.sink[h].double().expand(t, 1)], 1)
            z = torch.softmax(z, 1)[:, :n] @ v[h // (H // G)]
            out[t0:t0 + t, h] = z * torch.sigmoid(s.gate[t0:t0 + t, h].double()) if c["gate"] else z
        t0 += t
    return out
