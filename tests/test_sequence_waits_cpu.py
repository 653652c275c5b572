"""The roles of the kernels in csrc/decay.cu and csrc/window.cu as models: which of them waits for which, tile by tile, in every order that their speeds allow.

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


class Role(list):
    def wait(self, name, phase):
        self.append(("wait", name, phase, None))

    def arrive(self, name):
        self.append(("arrive", name, None, None))

    def commit(self, name):
        self.append(("commit", name, None, None))


def states_roles(tiles, stages):
    copy, products, operands = Role(), Role(), Role()
    for n in range(tiles):
        if n >= stages:
            copy.wait(f"free{n % stages}", n // stages - 1)
        copy.arrive(f"full{n % stages}")
        products.wait(f"full{n % stages}", n // stages)
        products.wait("split", n)
        products.commit("tails")
        products.commit(f"free{n % stages}")
        operands.wait(f"full{n % stages}", n // stages)
        if n:
            operands.wait("tails", n - 1)
        operands.arrive("split")
    products.commit("done")
    operands.wait("done", 0)
    return copy, products, operands


def grad_keys_roles(tiles, stages, ends):
    """ends: the tiles that hold the end of a sequence, whose rows behind it the weights' warps clear"""
    copy, products, rows = Role(), Role(), Role()
    copy.arrive("keys")
    products.wait("keys", 0)
    products.wait("full0", 0)
    products.commit("s")
    products.commit("dp")
    for n in range(tiles):
        if n >= stages:
            copy.wait(f"free{n % stages}", n // stages - 1)
        copy.arrive(f"full{n % stages}")
        more = n + 1 < tiles
        if more:
            products.wait(f"full{(n + 1) % stages}", (n + 1) // stages)
        products.wait("p", n)
        if more:
            products.commit("s")
        products.wait("ds", n)
        products.commit(f"free{n % stages}")
        products.commit("dp" if more else "done")
        if n in ends:
            rows.wait(f"full{n % stages}", n // stages)
            rows.wait("s", n)
            rows.wait("dp", n)
        rows.wait("s", n)
        rows.arrive("p")
        rows.wait("dp", n)
        rows.arrive("ds")
    rows.wait("done", 0)
    return copy, products, rows


def grad_queries_roles(tiles, slots):
    copy, products, rows = Role(), Role(), Role()
    copy.arrive("q")
    for x in range(2 * tiles):
        if x >= slots:
            copy.wait(f"free{x % slots}", x // slots - 1)
        copy.arrive(f"full{x % slots}")

    def scores(n):
        products.wait(f"full{2 * n % slots}", 2 * n // slots)
        products.commit(f"s{n % 2}")

    def values(n):
        x = 2 * n + 1
        products.wait(f"full{x % slots}", x // slots)
        products.commit("dp")
        products.commit(f"free{x % slots}")

    products.wait("q", 0)
    scores(0)
    values(0)
    if tiles > 1:
        scores(1)
    for n in range(tiles):
        products.wait("ds", n)
        if n + 1 < tiles:
            values(n + 1)
        products.commit(f"free{2 * n % slots}")
        if n + 1 == tiles:
            products.commit("done")
        if n + 2 < tiles:
            scores(n + 2)
        rows.wait(f"s{n % 2}", n // 2)
        if n + 1 == tiles:      # the end of the sequence
            rows.wait(f"full{2 * n % slots}", 2 * n // slots)
        rows.wait("dp", n)
        rows.arrive("ds")
    rows.wait("done", 0)
    return copy, products, rows


def window_roles(items, slots):
    """items: (tiles of keys, query tiles) of each"""
    copy, products, rows = Role(), Role(), (Role(), Role())
    x, done, scored, out = 0, [0, 0], [0, 0], [0, 0]
    for i, (keys, queries) in enumerate(items):
        if i:
            copy.wait("q_free", i - 1)
        copy.arrive("q")
        for y in range(x, x + 2 * keys):
            if y >= slots:
                copy.wait(f"free{y % slots}", y // slots - 1)
            copy.arrive(f"full{y % slots}")
        products.wait("q", i)
        products.wait(f"full{x % slots}", x // slots)
        for t in range(queries):
            products.commit(f"s{t}")
        products.commit(f"free{x % slots}")
        if keys == 1:
            products.commit("q_free")
        for j in range(keys):
            v, more = x + 2 * j + 1, j + 1 < keys
            products.wait(f"full{v % slots}", v // slots)
            if more:
                products.wait(f"full{(v + 1) % slots}", (v + 1) // slots)
            for t in range(queries):
                if j == 0 and done[t]:
                    products.wait(f"o_read{t}", done[t] - 1)
                products.wait(f"p{t}", scored[t])
                products.wait(f"p2{t}", scored[t])
                done[t] += not more
                products.commit(f"s{t}" if more else f"o{t}")
                rows[t].wait(f"s{t}", scored[t])
                if t == 0 and not more:
                    rows[t].wait(f"full{v % slots}", v // slots)
                rows[t].arrive(f"p{t}")
                rows[t].arrive(f"p2{t}")
                scored[t] += 1
            products.commit(f"free{v % slots}")
            if more:
                products.commit(f"free{(v + 1) % slots}")
            if j + 2 == keys:
                products.commit("q_free")
        for t in range(queries):
            rows[t].wait(f"o{t}", out[t])
            rows[t].arrive(f"o_read{t}")
            out[t] += 1
        x += 2 * keys
    return copy, products, *rows


def faults(progs):
    """The barriers that some order of the steps leaves a phase ahead of a role that waits for them, or a phase behind; 'stuck' where no role can go on."""
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
                if done[i] > phase + 1 or done[i] < phase:      # the parity of another phase
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
    assert faults(roles(tiles, stages, 2)) == set()


@pytest.mark.parametrize("progs", [states_roles(6, 2), states_roles(7, 4), grad_keys_roles(1, 2, {0}), grad_keys_roles(5, 2, {2, 4}), grad_keys_roles(7, 4, {3, 6}),
                                   grad_queries_roles(1, 5), grad_queries_roles(4, 5), grad_queries_roles(6, 8), window_roles([(1, 2), (2, 2), (1, 1), (3, 2)], 4),
                                   window_roles([(2, 1), (1, 2), (3, 2)], 8)],
                         ids=["states-2", "states-4", "keys-1", "keys-2", "keys-4", "queries-1", "queries-5", "queries-8", "window-4", "window-8"])
def test_no_barrier_of_the_other_kernels_does(progs):
    assert faults(progs) == set()


def test_the_model_sees_one_barrier_for_all_weights_run_ahead():
    """The weights of tile n + 1 need no step of the products behind A S of tile n: one barrier for all tiles would not do."""
    assert faults(roles(4, 2, 1)) >= {"weights0", "stuck"}


def test_the_kernel_has_the_barriers_of_the_model():
    """A barrier of the scores and one of the weights for even tiles, and one for odd."""
    import os
    import re
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "f3m_b200", "csrc", "decay.cu")) as f:
        code = f.read()
    body = code[code.index("decay_tiles(const"):code.index("decay_states(const")]
    assert re.search(r"wait\(b_weights_of\(n\), \(n >> 1\) & 1\)", body) and re.search(r"mbar_arrive\(b_weights_of\(n\)\)", body)
    assert re.search(r"all_wait\(b_score_of\(n\), \(n >> 1\) & 1\)", body)
