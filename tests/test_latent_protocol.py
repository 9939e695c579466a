"""Model checks of the latent attention kernels' mbarrier protocols
(csrc/latent.cu, csrc/latent_prefill.cu), on the CPU, with the scheduler of
test_ring_protocol.py: loads land in any order, the tensor core runs each
thread's operations in their order, warps run at any pace. Each role's loop is
restated with the parities of the source."""
import random
import re
from pathlib import Path

import pytest

from test_ring_protocol import Sim
from test_tree_protocol import watched


class Places:
    """Places of shared memory: what was loaded into each, whether it landed, and whether all its readers are done."""

    def __init__(self, sim):
        self.sim, self.held, self.landed, self.free = sim, {}, set(), {}

    def load(self, place, what, bar, parts=1):
        assert self.free.get(place, True), f"{what} overwrites {self.held[place]} in place {place} before it was read"
        self.held[place], self.free[place] = what, False
        self.landed.discard(place)

        def land():
            self.landed.add(place)
            self.sim.parts[bar] = self.sim.parts.get(bar, 0) + 1
            if self.sim.parts[bar] == parts:
                self.sim.parts[bar] = 0
                self.sim.arrive(bar)

        self.sim.loads.append(land)

    def read(self, place, what):
        assert self.held.get(place) == what and place in self.landed, \
            f"{what} read from place {place}, which holds {self.held.get(place)}"

    def done(self, place):
        self.free[place] = True


def tensor(sim, q, run):
    while True:
        yield ("tensor", q)
        op = sim.tqs[q].pop(0)
        if op[0] == "commit":
            sim.arrive(op[1])
        else:
            run(*op)


def simulate(sim, actors):
    sim.run({name: watched(sim, actor) for name, actor in actors.items()})


# ----------------------------------------------------------- absorbed form
def run_absorbed(seed, segments, warps, one_free_barrier=False):
    sim, rng = Sim(seed, 0), random.Random(seed + 1)
    sim.parts, sim.tqs = {}, {"s": [], "pv": []}
    kv, q = Places(sim), Places(sim)
    units = 3  # the rotated piece and pairs of latent ones (four in the kernel)
    for s in range(2):
        for u in range(units):
            sim.bar(f"Full{s}{u}"), sim.bar(f"Empty{s}{u}")
        sim.bar(f"SFull{s}"), sim.bar(f"SFree{s}", warps)
    sim.bar("PFull", warps), sim.bar("PVDone"), sim.bar("QFree"), sim.bar("OFree", warps)
    tiles = [(seg, t) for seg, n in enumerate(segments) for t in range(n)]
    last = {seg: sum(segments[:seg + 1]) - 1 for seg in range(len(segments))}
    s_buf, p_by, s_read, state = [None, None], {}, {}, {"pv": -1, "o": None}
    o_read = {}

    def producer():
        g = 0
        for seg, n in enumerate(segments):
            if seg:
                yield Sim.wait("QFree", (seg - 1) & 1, seg - 1)
            for t in range(n):
                stage = g & 1
                for u in range(units):
                    if g >= 2:
                        yield Sim.wait(f"Empty{stage}{u}", ((g >> 1) + 1) & 1, (g >> 1) - 1)
                    bar = f"Full{stage}{u}"
                    if t == 0:
                        q.load(u, (seg, u), bar, 2)
                    kv.load((stage, u), (g, u), bar, 2 if t == 0 else 1)
                    yield ("step",)
                g += 1

    def s_issuer():
        for g, (seg, _) in enumerate(tiles):
            stage = g & 1
            if g >= 2:
                if one_free_barrier:
                    yield Sim.wait("SFree0", (g - 2) & 1, g - 2)
                else:
                    yield Sim.wait(f"SFree{stage}", ((g >> 1) + 1) & 1, (g >> 1) - 1)
            for u in range(units):
                yield Sim.wait(f"Full{stage}{u}", (g >> 1) & 1, g >> 1)
                sim.tqs["s"].append(("S", g, u))
            sim.tqs["s"] += [("commit", f"SFull{stage}"), ("commit", f"Empty{stage}0")]
            if g == last[seg]:
                sim.tqs["s"].append(("commit", "QFree"))
            yield ("step",)

    def run_s(_, g, u):
        stage, seg = g & 1, tiles[g][0]
        kv.read((stage, u), (g, u))
        q.read(u, (seg, u))
        if u == 0:
            kv.done((stage, u))
            assert g < 2 or len(s_read[g - 2]) == warps, f"S of tile {g} over scores that are not read"
            s_buf[stage] = None
        if u == units - 1:
            s_buf[stage] = g
            if g == last[seg]:
                for v in range(units):
                    q.done(v)

    def pv_issuer():
        g = 0
        for seg, n in enumerate(segments):
            if seg:
                yield Sim.wait("OFree", (seg - 1) & 1, seg - 1)
            for _ in range(n):
                yield Sim.wait("PFull", g & 1, g)
                for u in range(1, units):
                    sim.tqs["pv"] += [("PV", g, u), ("commit", f"Empty{g & 1}{u}")]
                sim.tqs["pv"].append(("commit", "PVDone"))
                g += 1
                yield ("step",)

    def run_pv(_, g, u):
        kv.read((g & 1, u), (g, u))
        kv.done((g & 1, u))
        seg = tiles[g][0]
        assert len(p_by[g]) == warps and all(len(p_by.get(k, ())) == 0 for k in range(g + 1, len(tiles)))
        if g and tiles[g - 1][0] != seg:
            assert len(o_read[tiles[g - 1][0]]) == warps, "O restarts before it was read"
        if u == units - 1:
            assert state["pv"] == g - 1
            state["pv"] = g

    def rows(w):
        g = 0
        for seg, n in enumerate(segments):
            for t in range(n):
                yield Sim.wait(f"SFull{g & 1}", (g >> 1) & 1, g >> 1)
                assert s_buf[g & 1] == g, "scores of another tile"
                s_read.setdefault(g, set()).add(w)
                sim.arrive("SFree0" if one_free_barrier else f"SFree{g & 1}")
                yield ("step",)
                if g:
                    yield Sim.wait("PVDone", (g - 1) & 1, g - 1)
                    assert state["pv"] == g - 1, "P written or O rescaled beside a product"
                for u in range(1, units):
                    kv.read((g & 1, u), (g, u))  # repaired where it lies
                p_by.setdefault(g, set()).add(w)
                sim.arrive("PFull")
                g += 1
                yield ("step",)
            yield Sim.wait("PVDone", (g - 1) & 1, g - 1)
            assert state["pv"] == g - 1
            o_read.setdefault(seg, set()).add(w)
            sim.arrive("OFree")
            yield ("step",)

    actors = {"producer": producer(), "s_issuer": s_issuer(), "pv_issuer": pv_issuer(),
              "tensor_s": tensor(sim, "s", run_s), "tensor_pv": tensor(sim, "pv", run_pv)}
    actors.update({f"rows{w}": rows(w) for w in range(warps)})
    simulate(sim, actors)
    assert state["pv"] == len(tiles) - 1


def test_absorbed_protocol():
    rng = random.Random(1)
    for _ in range(300):
        segments = [rng.choice([1, 1, 2, 3, 5, 9]) for _ in range(rng.randint(1, 5))]
        run_absorbed(rng.randrange(1 << 30), segments, rng.randint(1, 4))


def test_the_scores_need_a_barrier_a_buffer():
    # One barrier for both: the rows may read two tiles' scores before the issuer looks, whose wait would then find the
    # parity of a phase to come.
    with pytest.raises(AssertionError, match="alias|two phases past|passes early|not read|deadlock"):
        for seed in range(80):
            run_absorbed(seed, [7, 2], 2, one_free_barrier=True)


def test_every_way_through_the_first_kernel_leaves_a_record():
    # The second kernel goes by the record of each CTA, and the scratch holds anything before: where shared memory is not
    # laid out as the roles need it, there is one with nothing to join.
    source = (Path(__file__).resolve().parents[1] / "nano-vllm-rs_b200" / "csrc" / "latent.cu").read_text()
    kernel = source[source.index("latent_kernel(const LatentParams p"):source.index("latent_join_kernel(")]
    unused = re.search(r"if \(!aligned\) \{(.*?)\n  \} else if \(warp == 0\)", kernel, re.S).group(1)
    record = "*reinterpret_cast<Join*>(part + 2 * kPartFloats) ="
    assert f"if (threadIdx.x == 128) {record} Join{{0, 0, 0, 0}};" in unused
    assert kernel.count(record) == 2  # and that of the rows' warps


# ----------------------------------------------------------- expanded form
SLOTS, K_PIECES, PIECES = 8, 3, 5


def run_expanded(seed, items, v_barriers=2):
    sim = Sim(seed, 0)
    sim.parts, sim.tqs = {}, {"s": [], "pv": []}
    ring, q = Places(sim), Places(sim)
    for s in range(SLOTS):
        sim.bar(f"Empty{s}")
    for s in range(v_barriers):
        sim.bar(f"VFull{s}"), sim.bar(f"VReady{s}")
    for s in range(2):
        for name in ("KFull", "QFull", "QFree", "SFull", "PFull", "PVDone", "ODone", "OFree", "StatsFull", "StatsFree",
                     "ItemFull"):
            sim.bar(f"{name}{s}")
        sim.bar(f"ItemEmpty{s}", 6)
    tiles = [(i, j) for i, n in enumerate(items) for j in range(max(n))]
    ready, s_of, p_of, pv_of = {}, [None, None], [None, None], [None, None]  # by query tile x: (item, tile)
    o_read, bad = {}, {}

    def take(i):
        return Sim.wait(f"ItemFull{i & 1}", (i >> 1) & 1, i >> 1)

    def producer():
        issued, gk, gv, used = 0, 0, 0, [0, 0]
        for i, n in enumerate(items):
            if i >= 2:
                yield Sim.wait(f"ItemEmpty{i & 1}", ((i >> 1) + 1) & 1, (i >> 1) - 1)
            assert i < 4 or bad[(i - 4) & 3] == "read", "the epilogue has not looked at what the mender left"
            bad[i & 3] = "new"
            sim.arrive(f"ItemFull{i & 1}")
            yield ("step",)
            order = []
            for j in range(max(n)):
                if j == 0:
                    order += [("K", 0, c) for c in range(3)] + [("Q", 0, 0), ("Q", 1, 0)]
                order += [("V", j, c) for c in range(2)]
                if j + 1 < max(n):
                    order += [("K", j + 1, c) for c in range(3)]
            for kind, j, c in order:
                if kind == "Q":
                    if n[j] == 0:
                        continue
                    if used[j]:
                        yield Sim.wait(f"QFree{j}", (used[j] - 1) & 1, used[j] - 1)
                    q.load(j, i, f"QFull{j}")
                    used[j] += 1
                    continue
                slot = issued % SLOTS
                if issued >= SLOTS:
                    yield Sim.wait(f"Empty{slot}", ((issued // SLOTS) + 1) & 1, issued // SLOTS - 1)
                bar = f"KFull{gk & 1}" if kind == "K" else f"VFull{gv % v_barriers}"
                ring.load(slot, (kind, i, j, c), bar, 3 if kind == "K" else 2)
                issued += 1
                gk += kind == "K" and c == 2
                gv += kind == "V" and c == 1
                yield ("step",)
        if len(items) >= 2:
            yield Sim.wait(f"ItemEmpty{len(items) & 1}", ((len(items) >> 1) + 1) & 1, (len(items) >> 1) - 1)

    def place(g, c):
        return (PIECES * g + c) % SLOTS

    def s_issuer():
        g, tx, ixq = 0, [0, 0], [0, 0]
        for i, n in enumerate(items):
            yield take(i)
            sim.arrive(f"ItemEmpty{i & 1}")
            for j in range(max(n)):
                yield Sim.wait(f"KFull{g & 1}", (g >> 1) & 1, g >> 1)
                for x in range(2):
                    if j >= n[x]:
                        continue
                    if j == 0:
                        yield Sim.wait(f"QFull{x}", ixq[x] & 1, ixq[x])
                    if tx[x]:
                        yield Sim.wait(f"PVDone{x}", (tx[x] - 1) & 1, tx[x] - 1)
                    sim.tqs["s"] += [("S", x, i, j, g), ("commit", f"SFull{x}")]
                    if j == n[x] - 1:
                        sim.tqs["s"] += [("qdone", x), ("commit", f"QFree{x}")]
                        ixq[x] += 1
                    tx[x] += 1
                for c in range(K_PIECES):
                    sim.tqs["s"] += [("done", place(g, c)), ("commit", f"Empty{place(g, c)}")]
                g += 1
                yield ("step",)

    def run_s(op, *a):
        if op == "done":
            ring.done(*a)
        elif op == "qdone":
            q.done(*a)
        else:
            x, i, j, g = a
            for c in range(K_PIECES):
                ring.read(place(g, c), ("K", i, j, c))
            q.read(x, i)
            assert p_of[x] is None or pv_of[x] == p_of[x], "S over a P that was not read"
            s_of[x] = (i, j)

    def pv_issuer():
        g, tx, ixo = 0, [0, 0], [0, 0]
        for i, n in enumerate(items):
            yield take(i)
            sim.arrive(f"ItemEmpty{i & 1}")
            for j in range(max(n)):
                yield Sim.wait(f"VReady{g % v_barriers}", (g // v_barriers) & 1, g // v_barriers)
                for x in range(2):
                    if j >= n[x]:
                        continue
                    if j == 0 and ixo[x]:
                        yield Sim.wait(f"OFree{x}", (ixo[x] - 1) & 1, ixo[x] - 1)
                    yield Sim.wait(f"PFull{x}", tx[x] & 1, tx[x])
                    sim.tqs["pv"] += [("PV", x, i, j, g), ("commit", f"PVDone{x}")]
                    if j == n[x] - 1:
                        sim.tqs["pv"].append(("commit", f"ODone{x}"))
                        ixo[x] += 1
                    tx[x] += 1
                for c in (3, 4):
                    sim.tqs["pv"] += [("done", place(g, c)), ("commit", f"Empty{place(g, c)}")]
                g += 1
                yield ("step",)

    def run_pv(op, *a):
        if op == "done":
            return ring.done(*a)
        x, i, j, g = a
        for c in (0, 1):
            ring.read(place(g, 3 + c), ("V", i, j, c))
        assert ready.get(g), "V that was not mended"
        assert p_of[x] == (i, j), "P of another tile"
        if j == 0 and any(items[k][x] for k in range(i)):
            before = max(k for k in range(i) if items[k][x])
            assert o_read.get((before, x)), "O restarts before it was read"
        pv_of[x] = (i, j)

    def mender():
        g = 0
        for i, n in enumerate(items):
            yield take(i)
            sim.arrive(f"ItemEmpty{i & 1}")
            for j in range(max(n)):
                yield Sim.wait(f"VFull{g % v_barriers}", (g // v_barriers) & 1, g // v_barriers)
                for c in (0, 1):
                    ring.read(place(g, 3 + c), ("V", i, j, c))
                ready[g] = True
                sim.arrive(f"VReady{g % v_barriers}")
                g += 1
                yield ("step",)

    def softmax(x):
        t = ix = 0
        for i, n in enumerate(items):
            yield take(i)
            sim.arrive(f"ItemEmpty{i & 1}")
            if n[x] == 0:
                continue
            for j in range(n[x]):
                yield Sim.wait(f"SFull{x}", t & 1, t)
                assert s_of[x] == (i, j)
                if j and sim.rng.random() < 0.3:
                    yield Sim.wait(f"PVDone{x}", (t - 1) & 1, t - 1)
                p_of[x] = (i, j)
                sim.arrive(f"PFull{x}")
                t += 1
                yield ("step",)
            if ix:
                yield Sim.wait(f"StatsFree{x}", (ix - 1) & 1, ix - 1)
            sim.arrive(f"StatsFull{x}")
            ix += 1
            yield ("step",)

    def epilogue():
        ixo = [0, 0]
        for i, n in enumerate(items):
            yield take(i)
            sim.arrive(f"ItemEmpty{i & 1}")
            for x in range(2):
                if n[x] == 0:
                    continue
                yield Sim.wait(f"StatsFull{x}", ixo[x] & 1, ixo[x])
                sim.arrive(f"StatsFree{x}")
                yield Sim.wait(f"ODone{x}", ixo[x] & 1, ixo[x])
                assert pv_of[x] == (i, n[x] - 1)
                o_read[i, x] = True
                sim.arrive(f"OFree{x}")
                ixo[x] += 1
                yield ("step",)
            bad[i & 3] = "read"

    simulate(sim, {"producer": producer(), "s_issuer": s_issuer(), "pv_issuer": pv_issuer(), "mender": mender(),
                   "softmax0": softmax(0), "softmax1": softmax(1), "epilogue": epilogue(),
                   "tensor_s": tensor(sim, "s", run_s), "tensor_pv": tensor(sim, "pv", run_pv)})
    assert len(ready) == len(tiles)


def _items(rng):
    items = []
    for _ in range(rng.randint(1, 6)):
        a = rng.choice([0, 1, 1, 2, 3, 6])
        kind = rng.random()
        items.append((a, a + 1) if kind < 0.5 else (a, a) if kind < 0.6 else (max(a, 1), 0) if kind < 0.8 else (0, rng.randint(0, 2)))
    return items


def test_expanded_protocol():
    rng = random.Random(2)
    for _ in range(300):
        run_expanded(rng.randrange(1 << 30), _items(rng))


def test_values_need_two_barriers():
    # With one, V of the next tile may land before the mender or the PV issuer has looked at this one's phase.
    with pytest.raises(AssertionError, match="alias|two phases past|passes early|deadlock"):
        rng = random.Random(3)
        for seed in range(100):
            run_expanded(seed, _items(rng), v_barriers=1)
