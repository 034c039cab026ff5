"""The stages of the 4-bit product of many rows, in every order in which its roles can run, on the CPU.

A barrier is the count of its completed phases; a wait for a parity ends while that count's last bit differs from it (PTX's mbarrier.try_wait.parity:
true for the phase before the current one). Roles: the warp that brings the tokens, two warps of each group that fill the weights (a phase of a stage is
full when both of the block's group and the tokens have arrived), the warp that issues the products, and the products, which are complete in their
order some time after they are issued. Reports of completed products arrive on their barriers later still, on different ones in any order."""
import ctypes

import pytest

from vosti_b200 import ops

TOKENS, WARPS = 0, 2


def schedule(tile, block):
    try:
        library = ops.library()
    except Exception as error:                       # no nvcc on this machine
        pytest.skip(f"the kernel library cannot be built here: {error}")
    out = (ctypes.c_int * 5)()
    assert library.vosti_gemm_int4_schedule(tile, block, out) == 0
    return dict(zip(("stages", "groups", "reports", "barrier", "parity"), out))


def rule_of(tile):
    rows = [schedule(tile, b) for b in range(40)]
    waits = [[(r["barrier"], r["parity"])] if r["barrier"] >= 0 else [] for r in rows]
    return rows[0]["stages"], rows[0]["groups"], [r["reports"] for r in rows], waits, waits


def explore(stages, groups, reports, fill_waits, token_waits, blocks):
    """None, or what goes wrong in some order: a role that waits for good, or a stage filled while its products still read it."""
    barriers = max(reports) + 1
    turns = [[b for b in range(blocks) if b % groups == g] for g in range(groups)]
    # a role's place is (blocks finished, waits of the next block passed): flat, so that a state is one tuple
    roles = [("tokens", None)] + [("fill", g) for g in range(groups) for _ in range(WARPS)] + [("issue", None), ("complete", None)]
    work = [list(range(blocks)) if r[0] != "fill" else turns[r[1]] for r in roles]
    issue, complete = len(roles) - 2, len(roles) - 1
    reported = [[b for b in range(blocks) if reports[b] == r] for r in range(barriers)]

    def moves(state):
        place, step, phases, arrived = state
        for i, (kind, _) in enumerate(roles):
            if place[i] == len(work[i]):
                continue
            b = work[i][place[i]]
            s = b % stages
            if kind in ("tokens", "fill"):
                waits = (token_waits if kind == "tokens" else fill_waits)[b]
                if step[i] < len(waits):
                    barrier, parity = waits[step[i]]
                    if (phases[barrier] & 1) != parity:
                        yield place, step[:i] + (step[i] + 1,) + step[i + 1:], phases, arrived
                    continue
                if b >= stages and place[complete] <= b - stages:
                    raise AssertionError(f"stage {s} is filled for block {b} before block {b - stages} is complete")
                count = arrived[s] + 1
                full = count == WARPS + 1
                yield (place[:i] + (place[i] + 1,) + place[i + 1:], step[:i] + (0,) + step[i + 1:],
                       phases[:barriers + s] + (phases[barriers + s] + full,) + phases[barriers + s + 1:], arrived[:s] + (0 if full else count,) + arrived[s + 1:])
            elif kind == "issue":
                if (phases[barriers + s] & 1) != ((b // stages) & 1):
                    yield place[:i] + (place[i] + 1,) + place[i + 1:], step, phases, arrived
            elif place[issue] > b:
                yield place[:i] + (place[i] + 1,) + place[i + 1:], step, phases, arrived
        for r in range(barriers):
            if phases[r] < len(reported[r]) and reported[r][phases[r]] < place[complete]:
                yield place, step, phases[:r] + (phases[r] + 1,) + phases[r + 1:], arrived
    start = ((0,) * len(roles), (0,) * len(roles), (0,) * (barriers + stages), (0,) * stages)
    seen, todo = {start}, [start]
    while todo:
        state = todo.pop()
        try:
            following = list(moves(state))
        except AssertionError as wrong:
            return str(wrong)
        if not following and any(p < len(w) for p, w in zip(state[0], work)):
            return f"every role waits for good: {[(r, w[p] if p < len(w) else 'ended') for r, p, w in zip(roles, state[0], work)]}"
        for new in following:
            if new not in seen:
                seen.add(new)
                todo.append(new)
    return None


@pytest.mark.parametrize("tile", range(4))
def test_no_order_of_the_roles_stops_or_overwrites(tile):
    stages, groups, reports, fill, tokens = rule_of(tile)
    assert explore(stages, groups, reports, fill, tokens, 4 * stages * groups + 1) is None


def test_the_model_finds_faults():
    """Two groups over three stages with one report a stage: a wait that another group's block can overtake stops, and without it a stage is overwritten."""
    parity = lambda b: (b // 3) & 1
    reports, tokens = [b % 3 for b in range(20)], [[(b % 3, parity(b - 3))] if b >= 3 else [] for b in range(20)]
    overtaken = [([((b - 1) % 3, parity(b - 4))] if b > 3 else []) + w for b, w in enumerate(tokens)]
    assert "waits for good" in explore(3, 2, reports, overtaken, tokens, 9)
    assert "filled" in explore(3, 2, reports, tokens, tokens, 9)
