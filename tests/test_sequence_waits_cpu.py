"""The roles of decay_tiles (csrc/decay.cu) as a model: which of them waits for which, tile by tile, in every order that their speeds allow.

A wait names a phase's parity only, so a barrier must not complete phase n + 1 while a role may still be waiting for phase n: the role
would find the parity of n again and wait until its limit.  The model's steps are those of the kernel, in its order; the tensor
cores complete what is committed to them in order, at any later time.
"""
import pytest


def roles(tiles, stages, weights_barriers):
    """Each role's steps: (wait | arrive | commit | test, barrier, phase of that barrier, None or the outcome of the last test that the step needs)"""
    score = lambda n: (f"score{n % 2}", n // 2)  # noqa: E731
    weights = lambda n: (f"weights{n % weights_barriers}", n // weights_barriers)  # noqa: E731
    full = lambda n: (f"full{n % stages}", n // stages)  # noqa: E731
    free = lambda n: (f"free{n % stages}", n // stages)  # noqa: E731
    copy, products, rows, operands = [], [], [], []
    step = lambda to, kind, bar, need=None: to.append((kind, *bar, need))  # noqa: E731

    for n in range(tiles):
        if n >= stages:
            step(copy, "wait", free(n - stages))
        step(copy, "arrive", full(n))

    def scores(n, need):
        step(products, "wait", full(n), need)
        step(products, "commit", score(n), need)

    scores(0, None)
    for n in range(tiles):
        if n:
            step(products, "wait", ("read", n - 1))
        step(products, "wait", ("state", n))
        step(products, "commit", ("inter", n))
        if n + 1 < tiles:
            step(products, "test", full(n + 1))
            scores(n + 1, True)
        step(products, "wait", ("split", n))
        step(products, "commit", ("moved", n))
        step(products, "wait", weights(n))
        step(products, "wait", ("scaled", n))
        step(products, "commit", ("done", n))
        step(products, "commit", free(n))
        if n + 1 < tiles:
            scores(n + 1, False)

    def weigh(n, need):
        step(rows, "wait", score(n), need)
        step(rows, "arrive", weights(n), need)

    weigh(0, None)
    for n in range(tiles):
        step(rows, "wait", ("inter", n))
        step(rows, "arrive", ("scaled", n))
        if n + 1 < tiles:
            step(rows, "test", score(n + 1))
            weigh(n + 1, True)
        step(rows, "wait", ("done", n))
        step(rows, "arrive", ("read", n))
        if n + 1 < tiles:
            weigh(n + 1, False)

    for n in range(tiles + 1):
        if n < tiles:
            step(operands, "wait", full(n))
            step(operands, "wait", score(n))
        if n:
            step(operands, "wait", ("moved", n - 1))
        if n < tiles:
            step(operands, "arrive", ("state", n))
            step(operands, "wait", ("inter", n))
            step(operands, "arrive", ("split", n))
    return copy, products, rows, operands


def faults(tiles, stages, weights_barriers):
    """The barriers that some order of the steps leaves a phase ahead of a role that waits for them; 'stuck' where no role can go on."""
    progs = roles(tiles, stages, weights_barriers)
    names = sorted({s[1] for p in progs for s in p})
    at = {n: i for i, n in enumerate(names)}
    start = ((0,) * len(progs), (False,) * len(progs), (0,) * len(names), ())
    seen, todo, found = {start}, [start], set()
    while todo:
        pcs, flags, done, queue = todo.pop()
        after = []

        def completed(i):
            return done[:i] + (done[i] + 1,) + done[i + 1:]

        if queue:      # the tensor cores complete the oldest commit
            after.append((pcs, flags, completed(queue[0]), queue[1:]))
        for r, prog in enumerate(progs):
            if pcs[r] == len(prog):
                continue
            kind, name, phase, need = prog[pcs[r]]
            i, on = at[name], pcs[:r] + (pcs[r] + 1,) + pcs[r + 1:]
            if need is not None and need != flags[r]:
                after.append((on, flags, done, queue))
            elif kind == "wait":
                if done[i] > phase + 1:
                    found.add(name)
                if done[i] == phase + 1:
                    after.append((on, flags, done, queue))
            elif kind == "test":
                after.append((on, flags[:r] + (done[i] == phase + 1,) + flags[r + 1:], done, queue))
            elif kind == "arrive":
                after.append((on, flags, completed(i), queue))
            else:
                after.append((on, flags, done, queue + (i,)))
        if not after and any(pc < len(p) for pc, p in zip(pcs, progs)):
            found.add("stuck")
        for s in after:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return found


@pytest.mark.parametrize("tiles,stages", [(1, 2), (5, 2), (5, 3), (6, 4)])
def test_no_barrier_of_decay_tiles_runs_ahead_of_a_role_that_waits(tiles, stages):
    assert faults(tiles, stages, 2) == set()


def test_the_model_sees_one_barrier_for_all_weights_run_ahead():
    """The weights of tile n + 1 need no step of the products behind A S of tile n: one barrier for all tiles would not do."""
    assert faults(4, 2, 1) >= {"weights0", "stuck"}


def test_the_kernel_has_the_barriers_of_the_model():
    """A barrier of the scores and one of the weights for even tiles, and one for odd."""
    import os
    import re
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "f3m_b200", "csrc", "decay.cu")) as f:
        code = f.read()
    body = code[code.index("decay_tiles(const"):code.index("decay_states(const")]
    assert re.search(r"wait\(b_weights_of\(n\), \(n >> 1\) & 1\)", body) and re.search(r"mbar_arrive\(b_weights_of\(n\)\)", body)
    assert re.search(r"all_wait\(b_score_of\(n\), \(n >> 1\) & 1\)", body)
