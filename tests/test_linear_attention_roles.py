"""CPU: the order of the roles in the bf16 prompt kernel of linear attention
(prompt_direct_kernel), as a graph of what each role waits for, issues and
signals. Whatever the speed of its warps, no buffer may be written before all
that reads it is done, and no wait may come after its barrier's next phase.

The rings' sizes and the loading warp's waits are read from the source; the
rest restates the roles in its comments.
"""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "mamba-onnx_b200" / "csrc" /
          "linear_attention_mma.cu").read_text()
CHUNKS = 14


def rings():
    """Barriers of DirectSmall and how many chunks use different ones."""
    body = re.search(r"struct __align__\(16\) DirectSmall \{(.*?)\n\};", SOURCE, re.S).group(1)
    found = {}
    for line in re.findall(r"uint64_t ([^;]*);", body):
        for name in line.split(","):
            m = re.fullmatch(r"\s*(\w+)(?:\[(\d+)\])?\s*", name)
            found[m.group(1)] = int(m.group(2) or 1)
    return found


def loader_waits():
    """Which barriers the loading warp waits for before q's and k and v's tiles
    are loaded again, in order."""
    role = SOURCE[SOURCE.index("warp == 19)"):SOURCE.index("state group", SOURCE.index("warp == 19)"))]
    loop = role[role.index("for (int c = -2;"):]
    q = loop.index("load_q(c + 2)")
    kv = loop.index("load_kv(c + kStages)")
    waits = [(m.start(), m.group(1)) for m in re.finditer(r"wait\(&s\.(\w+)\[", loop)]
    return [n for at, n in waits if at < q], [n for at, n in waits if q < at < kv]


class Graph:
    def __init__(self):
        self.before = {}     # event -> events that precede it
        self.waits = []      # (event, barrier, chunk)

    def role(self, name):
        last = [None]

        def event(what, chunk, *also):
            e = (name, what, chunk)
            while e in self.before:  # (a wait that a role repeats)
                e = (name, e[1] + " again", chunk)
            self.before[e] = set(also) | ({last[0]} if last[0] else set())
            last[0] = e
            return e

        def wait(bar, chunk):
            e = event("wait " + bar, chunk, ("done", bar, chunk))
            self.waits.append((e, bar, chunk))
            return e

        def signal(bar, chunk):  # this role's arrival, or what it issued being done
            self.before.setdefault(("done", bar, chunk), set()).add(event("signal " + bar, chunk))

        return event, wait, signal

    def ancestors(self):
        """Events known to precede each event; raises on a cycle."""
        known, active = {}, set()

        def visit(e):
            if e not in known:
                assert e not in active, f"{e} waits for itself"
                active.add(e)
                known[e] = set()
                for b in self.before.get(e, ()):
                    known[e] |= visit(b) | {b}
                active.discard(e)
            return known[e]

        for e in list(self.before):
            visit(e)
        return known


def kernel(aggregate, n=CHUNKS):
    g = Graph()
    emits, wait_q, wait_kv = not aggregate, *loader_waits()
    event, wait, signal = g.role("load")
    for c in range(min(2, n) if emits else 0):
        signal("q_full", c)
    for c in range(min(3, n)):
        signal("full", c)
    for c in range(-2, n):
        if c + 2 < n:
            event("write decays", c + 2)
            signal("decays", c + 2)
        if c < 0 or c + 1 == n:
            continue
        if emits and c + 2 < n:
            for bar in wait_q:
                wait(bar, c)
            signal("q_full", c + 2)
        for bar in wait_kv:
            if emits or bar == "ds":
                wait(bar, c)
        if c + 3 < n:
            signal("full", c + 3)

    event, wait, signal = g.role("dS")
    for c in range(n):
        wait("full", c)
        back = 1 if emits else 2
        if c >= back:
            wait("ds_read", c - back)
        wait("v_ready", c)
        signal("ds", c)

    def weigh_values(event, wait, signal, c):
        wait("decays", c)
        wait("full", c)
        event("write values", c)
        signal("v_ready", c)

    if emits:
        event, wait, signal = g.role("O")
        for c in range(n):
            wait("q_full", c)
            wait("full", c)
            if c > 0:
                wait("o_read", c - 1)
            wait("s_ready", c)
            signal("o1", c)
            wait("p_ready", c)
            signal("out", c)
        event, wait, signal = g.role("scores")
        for c in range(n):
            wait("q_full", c)
            wait("full", c)
            if c > 0:
                wait("p_ready", c - 1)
            signal("scores", c)

        def weigh_scores(event, wait, signal, c):
            wait("decays", c)
            wait("scores", c)
            event("write P", c)
            signal("p_ready", c)

        event, wait, signal = g.role("lower outputs")
        weigh_scores(event, wait, signal, 0)
        for c in range(n):
            if c + 1 < n:
                weigh_scores(event, wait, signal, c + 1)
            wait("out", c)
            signal("o_read", c)
        event, wait, signal = g.role("upper outputs")
        for c in range(n):
            wait("out", c)
            signal("o_read", c)
    else:
        event, wait, signal = g.role("values")
        for c in range(n):
            if c >= 2:
                wait("ds", c - 2)
            weigh_values(event, wait, signal, c)

    event, wait, signal = g.role("state")
    if emits:
        weigh_values(event, wait, signal, 0)
        event("write S", 0)
        signal("s_ready", 0)
    for c in range(n):
        wait("decays", c)
        wait("ds", c)
        if emits and c + 1 < n:
            weigh_values(event, wait, signal, c + 1)
        signal("ds_read", c)
        if emits and c + 1 < n:
            wait("o1", c)
            event("write S", c + 1)
            signal("s_ready", c + 1)
    return g


@pytest.mark.parametrize("aggregate", [False, True])
def test_buffers_are_written_after_their_readers(aggregate):
    known = kernel(aggregate).ancestors()
    # (write, chunks later): what has to be done with the buffer by then
    rules = {("load", "signal full", 3): [("done", "ds")]}
    if aggregate:
        rules[("values", "write values", 2)] = [("done", "ds")]
        rules[("dS", "signal ds", 2)] = [("done", "ds_read")]
        rules[("load", "write decays", 8)] = [("values", "write values"), ("state", "signal ds_read")]
    else:
        rules[("load", "signal full", 3)] += [("done", "out"), ("done", "scores")]
        rules[("load", "signal q_full", 2)] = [("done", "o1"), ("done", "scores")]
        rules[("lower outputs", "write P", 2)] = [("done", "out")]
        rules[("scores", "signal scores", 1)] = [("lower outputs", "write P")]
        rules[("O", "signal o1", 1)] = [("done", "o_read")]
        rules[("dS", "signal ds", 1)] = [("done", "ds_read")]
        rules[("state", "write values", 1)] = [("done", "ds")]
        rules[("state", "write S", 1)] = [("done", "o1")]
        rules[("load", "write decays", 8)] = [("done", "o_read"), ("lower outputs", "write P"),
                                              ("state", "signal ds_read"), ("state", "write values")]
    for (role, what, later), readers in rules.items():
        checked = 0
        for c in range(CHUNKS - later):
            write = (role, what, c + later)
            for reader in readers:
                assert (*reader, c) in known[write], f"{write} does not wait for {(*reader, c)}"
                checked += 1
        assert checked


def test_q_tiles_are_waited_for_before_they_land_again():
    """A waiter sees a barrier's phase only until the ring's next one is done."""
    g = kernel(False)
    known = g.ancestors()
    for e, bar, c in g.waits:
        if bar == "q_full" and c + rings()[bar] < CHUNKS:
            assert e in known[("done", bar, c + rings()[bar])], f"{e} may come a phase late"


@pytest.mark.parametrize("aggregate", [False, True])
def test_no_wait_comes_a_phase_late(aggregate):
    """The same for every barrier: with parities a waiter that comes after the
    ring's next completion would wait for the one after that."""
    g = kernel(aggregate)
    known = g.ancestors()
    for e, bar, c in g.waits:
        if c + rings()[bar] < CHUNKS:
            assert e in known.get(("done", bar, c + rings()[bar]), {e}), f"{e} may come a phase late"
