"""The hand-overs between the warp roles of the distillation kernel, as a model that is searched
through whatever order its steps come in, on the CPU.

A role is a list of steps.  `wait` is an mbarrier's parity wait (bounded on the device: once a wait
has run out every later one returns at once, here `abort`), `arrive` its arrival; `sync` and `signal`
are a barrier that counts threads, whose wait nothing bounds.  `done` checks that every compute warp
has left the row.
"""
from pathlib import Path

import pytest

WARPS = 2  # compute warps of the model


def roles(live, counted):
    """(roles, arrivals a phase needs) of a CTA walking the rows `live` (False: masked).  counted:
    compute and finisher meet at a barrier that counts threads; else by the mbarrier `stored`."""
    teacher, compute, finisher, loader = [], [], [], []
    for it, on in enumerate(live):
        b, ph = it & 1, (it >> 1) & 1
        loader += [("wait", "left", (it & 1) ^ 1), ("arrive", "full")]
        teacher += [("wait", f"done{b}", ph ^ 1), ("wait", "full", it & 1), ("arrive", f"ready{b}")]
        compute += [("wait", f"ready{b}", ph)]
        if on:
            compute += [("wait", "full", it & 1), ("sync", "compute")]
        compute += [("arrive", "left")]
        finisher += [("wait", f"ready{b}", ph)]
        if counted:
            compute += [("signal", "row")] * on + [("arrive", f"done{b}")]
            finisher += [("sync", "row"), ("done", it)] * on + [("arrive", f"done{b}")]
        else:
            compute += [("arrive", f"stored{b}")]
            finisher += [("wait", f"stored{b}", ph), ("done", it), ("arrive", f"done{b}")]
    need = {"left": WARPS, "full": 1, "compute": WARPS, "row": WARPS + 1}
    for b in (0, 1):
        need.update({f"ready{b}": 1, f"stored{b}": WARPS, f"done{b}": WARPS + 1 if counted else 1})
    return [teacher, finisher, loader] + [compute] * WARPS, need


def search(live, counted, abort):
    """Every order of the steps: what can go wrong, or None.  abort: the waits may give up at any time."""
    procs, need = roles(live, counted)
    names = sorted(need)
    slot = {n: i for i, n in enumerate(names)}
    last = [j for j, s in enumerate(procs[-1]) if s[0] in ("signal", "arrive")]
    ends = []  # compute's step that ends each row
    for it in range(len(live)):
        tail = [j for j in last if procs[-1][j][1] in (("stored%d" % (it & 1)), ("done%d" % (it & 1)))]
        ends.append(tail[it >> 1])
    start = (tuple([0] * len(procs)), tuple([0] * len(names)), tuple([-1] * len(procs)), False)
    seen, todo = {start}, [start]
    while todo:
        at, arrived, waiting, gone = todo.pop()
        moves = []
        for p, steps in enumerate(procs):
            if at[p] == len(steps):
                continue
            step = steps[at[p]]
            a, w, forward = list(arrived), list(waiting), True
            if step[0] == "wait":
                phase = arrived[slot[step[1]]] // need[step[1]]
                if not gone and (phase & 1) == step[2]:
                    continue
            elif step[0] == "done":
                late = [c for c in range(3, len(procs)) if at[c] <= ends[step[1]] - counted]
                if late and not gone:
                    return f"the finisher takes row {step[1]} before compute has left it"
            elif step[0] == "sync":
                i = slot[step[1]]
                if waiting[p] < 0:
                    a[i] += 1
                    w[p] = arrived[i] // need[step[1]]
                    forward = False
                elif arrived[i] // need[step[1]] > waiting[p]:
                    w[p] = -1
                else:
                    continue
            else:
                a[slot[step[1]]] += 1
            moves.append((tuple(x + (forward and q == p) for q, x in enumerate(at)), tuple(a), tuple(w), gone))
        if not moves and any(x < len(s) for x, s in zip(at, procs)):
            return "no role can go on"
        if abort and not gone:
            moves.append((at, arrived, waiting, True))
        for m in moves:
            if m not in seen:
                seen.add(m)
                todo.append(m)
    return None


ROWS = [[True] * 5, [True, False, True, True, False], [False, True, False, False, True]]


@pytest.mark.parametrize("live", ROWS)
def test_rows_are_handed_over_in_order(live):
    assert search(live, counted=False, abort=False) is None


@pytest.mark.parametrize("live", [r[:4] for r in ROWS])
def test_a_wait_that_gives_up_ends_the_kernel(live):
    assert search(live, counted=False, abort=True) is None


def test_the_model_sees_a_barrier_without_back_pressure():
    """With a barrier that counts threads, compute's arrival for the next row stands in for the
    finisher's for this one; and after a wait has given up, nothing ends the finisher's."""
    assert search([True] * 4, counted=True, abort=False) is not None
    assert search([True] * 4, counted=True, abort=True) is not None


def test_roles_meet_at_bounded_waits_only():
    csrc = Path(__file__).resolve().parents[1] / "autokernel-halo-strix_b200" / "csrc"
    text = (csrc / "distill.cu").read_text()
    assert "bar.arrive" not in text
    assert text.count("bar.sync") == 1 and text.count("compute_sync(kCompute)") == 1
