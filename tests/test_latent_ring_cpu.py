"""The order in which the prompts' kernel fills its ring of key and value chunks (csrc/latent_ring.cuh),
run on the host and checked against everything that waits for it.

The header's order is compiled into a host program that writes down what the producer does: its waits
and its copies.  The other roles -- the warp that issues S = Q K^T, the one that issues P V, the
two softmax warpgroups -- are written here as the kernel has them.  All of it becomes one graph of
"comes before": program order in each role, and from what completes a phase of a barrier to whoever
waits for it.  Two things have to follow from the graph alone, whatever anything takes:

* a barrier is waited for by parity, so a phase may be announced or waited for only when the phase before
  it is complete, and complete only when all waits for the phase before it are over;
* a copy may land in a chunk only when the products that read what was there are complete."""

import subprocess
from pathlib import Path

import pytest

from _phases import Graph

CSRC = Path(__file__).resolve().parents[1] / "vllm-nt_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "latent_ring.cuh"
struct Ops {
  bool keys_half_used(unsigned g) { std::printf("wait KEmpty %u\n", g); return true; }
  bool keys_used(unsigned g) { std::printf("wait KDone %u\n", g); return true; }
  bool values_used(unsigned g) { std::printf("wait VEmpty %u\n", g); return true; }
  void load_keys(unsigned g) { std::printf("load K %u\n", g); }
  void load_values(unsigned g) { std::printf("load V %u\n", g); }
};
int main(int, char** argv) {
  using namespace ntb200;
  const unsigned tiles = std::atoi(argv[1]);
  for (unsigned g = 0; g < tiles; ++g) {
    std::printf("chunks K %u", g);
    for (unsigned c = 0; c < kRingKeys; ++c) std::printf(" %u", (k_chunk(g) + c) % kRingChunks);
    std::printf("\nchunks V %u", g);
    for (unsigned c = 0; c < kRingValues; ++c) std::printf(" %u", (v_chunk(g) + c) % kRingChunks);
    std::printf("\n");
  }
  Ops ops;
  RingFill fill;
  for (unsigned g = 0; g < tiles; ++g) {
    fill.keys(ops);
    fill.values_behind(ops);
  }
  fill.last_values(ops);
}
"""


@pytest.fixture(scope="module")
def producer(tmp_path_factory):
    """tiles -> (what the producer does, the chunks of every copy)"""
    where = tmp_path_factory.mktemp("ring")
    (where / "order.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(where / "order.cpp"), "-o", str(where / "order")], check=True)

    def run(tiles):
        lines = subprocess.run([str(where / "order"), str(tiles)], check=True, capture_output=True, text=True).stdout.split("\n")
        words = [line.split() for line in lines if line]
        chunks = {(w[1], int(w[2])): [int(c) for c in w[3:]] for w in words if w[0] == "chunks"}
        return [(w[0], w[1], int(w[2])) for w in words if w[0] != "chunks"], chunks

    return run


# Barriers are named by the tiles that they count (the phase after tile g's is tile g + 2's: even and odd
# tiles), or by tile A and B of the rows.


def step(bar):
    return 2 if isinstance(bar, str) and bar[0] in "KV" else 1


def build(trace, items):
    """The graph of one CTA that works on items of (key tiles of rows A, of rows B)."""
    g = Graph(step)
    done = lambda bar, n: ("done", bar, n)  # noqa: E731

    last = None
    for i, (what, which, n) in enumerate(trace):  # the producer
        if what == "wait":
            last = g.wait(which, n, "producer", last)
        else:
            last = g.event(("set", which + "Full", n), last)
            g.event(("copy", which, n), last)
            g.event(done(which + "Full", n), last)

    tiles = [max(item) for item in items]
    base = [sum(tiles[:i]) for i in range(len(items))]
    product = {}  # (rows, index among the rows' own) -> number among all S products
    last, ns, count = None, 0, [0, 0]
    for item, b, n in zip(items, base, tiles):  # S = Q K^T
        for j in range(n):
            last = g.wait("KFull", b + j, "S", last)
            for x in (0, 1):
                if j >= item[x]:
                    continue
                if ns > 0:
                    last = g.wait("SFree", ns - 1, "S", last)
                last = g.event(("issue S", ns), last)
                # a commit completes when everything issued before it has
                if x == 1 or j >= item[1]:
                    g.event(done("KEmpty", b + j), last)
                    g.event(done("KDone", b + j), last, done("KEmpty", b + j))
                g.event(done(("SFull", x), count[x]), last)
                product[x, count[x]] = ns
                count[x] += 1
                ns += 1
    last, count, begun, pv = None, [0, 0], [0, 0], None
    for item, b, n in zip(items, base, tiles):  # O += P V
        for j in range(n):
            last = g.wait("VFull", b + j, "PV", last)
            for x in (0, 1):
                if j >= item[x]:
                    continue
                if j == 0 and begun[x] > 0:
                    last = g.wait(("OFree", x), begun[x] - 1, "PV", last)
                last = g.wait(("PFull", x), count[x], "PV", last)
                pv = g.event(done(("PvDone", x), count[x]), last, pv)
                if x == 1 or j >= item[1]:
                    g.event(done("VEmpty", b + j), pv)
                begun[x] += j == 0
                count[x] += 1
    for x in (0, 1):  # the softmax of each tile of rows
        last, idx, begun = None, 0, 0
        for item in items:
            for j in range(item[x]):
                last = g.wait(("SFull", x), idx, "softmax", last)
                g.event(done("SFree", product[x, idx]), last)
                if j > 0:
                    last = g.wait(("PvDone", x), idx - 1, "softmax", last)
                last = g.event(("weights", x, idx), last)
                g.event(done(("PFull", x), idx), last)
                idx += 1
            if item[x] > 0:
                last = g.wait(("PvDone", x), idx - 1, "softmax", last)
                g.event(done(("OFree", x), begun), last)
                begun += 1
    return g


def faults(trace, chunks, items):
    g = build(trace, items)
    anc = g.ancestors()
    found = g.faults(anc)
    # (chunk, in the order of their copies) -> what is in it
    inside = {}
    for what, which, n in trace:
        if what != "load":
            continue
        for i, c in enumerate(chunks[which, n]):
            if c in inside:
                kind, m, part = inside[c]
                read = ("done", "VEmpty", m) if kind == "V" else ("done", "KEmpty" if part < 2 else "KDone", m)
                if read not in anc["set", which + "Full", n]:
                    found.append(f"{which} {n} lands on {kind} {m}")
            inside[c] = (which, n, i)
    return found


ITEMS = [
    [(1, 0)], [(2, 0)], [(3, 0)], [(4, 0)], [(7, 0)],            # at most 128 rows
    [(0, 1)], [(0, 5)],                                          # only the second rows see keys
    [(1, 2)], [(3, 4)], [(4, 5)], [(8, 9)],                      # causal: the second rows see one tile more
    [(2, 2)], [(5, 5)], [(6, 6)],
    [(5, 6), (3, 4), (1, 2)], [(1, 0), (1, 0), (1, 0), (1, 0)],  # several items a CTA
    [(5, 5), (3, 0)], [(6, 6), (0, 4), (0, 0), (2, 0)], [(0, 0)], [(3, 0), (0, 0), (4, 5)],
]


@pytest.mark.parametrize("items", ITEMS, ids=str)
def test_the_ring_is_filled_safely(producer, items):
    trace, chunks = producer(sum(max(i) for i in items))
    assert [e for e in trace if e[0] == "load" and e[1] == "K"] == [("load", "K", g) for g in range(sum(max(i) for i in items))]
    assert len([e for e in trace if e[:2] == ("load", "V")]) == sum(max(i) for i in items)
    assert faults(trace, chunks, items) == []


def test_the_check_sees_a_missing_wait(producer):
    """With any of the producer's waits left out of the trace some item shows it."""
    tiles = {str(items): producer(sum(max(i) for i in items)) for items in ITEMS}
    for kind in ("KEmpty", "KDone", "VEmpty"):
        assert any(faults([e for e in trace if e[:2] != ("wait", kind)], chunks, items)
                   for items in ITEMS for trace, chunks in [tiles[str(items)]])
    # the wait before the last values alone: one tile of rows and three key tiles, or one tile more for the second rows
    for items in ([(3, 0)], [(4, 5)]):
        trace, chunks = tiles[str(items)]
        at = max(i for i, e in enumerate(trace) if e[:2] == ("wait", "VEmpty"))
        assert trace[at][2] == sum(max(i) for i in items) - 3
        assert any("VFull" in f for f in faults(trace[:at] + trace[at + 1 :], chunks, items))
