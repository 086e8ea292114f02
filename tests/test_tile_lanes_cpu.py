"""Instructions that a whole warp has to come to together (loads and stores of tensor memory, barriers of some warps) in the kernel of 8-bit cache portions: between the last
branch that lanes take by numbers of their own and each of them stands something that joins the lanes again, a vote or an exchange between all of them.  A loop is read
twice, so that what parts the lanes at its end is seen ahead of its beginning."""
import re

import test_step_launch_cpu as steps

PARTS = r"\bif \((?:lane|tid|r|mx|most_v|part)\b"                                                   # by a lane's place, row, scores
JOINS = r"(?<!&& )(?<!&& !)\b(?:warp_meet|wait_long|__(?:any|all|ballot|shfl\w*)_sync)\("             # (behind && they may be left out)
TOGETHER = r"\b(?:tmem_(?:load|store)\d+|tmem_wait_st|bar_sync)\("


def apart(text):
    """calls that lanes may come to apart"""
    joined, bad = True, []
    for m in re.finditer(f"(?P<parts>{PARTS})|(?P<joins>{JOINS})|(?P<together>{TOGETHER})", text):
        if m.lastgroup == "together" and not joined:
            bad.append(text[m.start():text.index(";", m.start())])
        joined = joined if m.lastgroup == "together" else m.lastgroup == "joins"
    return bad


def block(text, at):
    i = text.index("{", at)
    depth, k = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(text[k], 0)
        if depth == 0:
            return text[i:k + 1]
        k += 1


def test_the_check_itself():
    assert apart("if (lane == 0) x(); bar_sync(3, 4);") == ["bar_sync(3, 4)"]
    assert apart("if (r < n) x(); warp_meet(); bar_sync(3, 4);") == []
    assert apart("if (mx > m) x(); if (k >= 2 && !wait_long(b)) y(); tmem_store8(t, v);") == ["tmem_store8(t, v)"]
    assert apart(2 * "tmem_load16(t, v); if (r >= rows) continue; ") == ["tmem_load16(t, v)"]


def test_lanes_are_together():
    body = {n: b for (_, n), (_, b) in steps.kernels().items()}["kv8_tile_kernel"]
    body = re.sub(r"\s+", " ", body[body.index("more_registers"):])  # the warps of weights
    found = set(apart(body))
    loops = [block(body, m.start()) for m in re.finditer(r"\bfor \(", body) if "{" in body[m.start():m.start() + 120]]
    assert len(loops) > 5
    for loop in loops:
        if re.search(TOGETHER, loop):
            found |= set(apart(loop + loop))
    assert not found, found
