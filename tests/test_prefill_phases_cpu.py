"""The waits of the paged prefill's roles, with the phases that tell a product's end taken from
csrc/prefill_phases.cuh: each of them has to be right whatever anything takes (see _phases.py)."""

import itertools
import subprocess
from pathlib import Path

import pytest

from _phases import Graph

CSRC = Path(__file__).resolve().parents[1] / "vllm-nt_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "prefill_phases.cuh"
int main() {
  for (unsigned g = 0; g < 64; ++g)
    std::printf("%u %u\n", ntb200::product_phase(g).barrier, ntb200::product_phase(g).parity);
}
"""


@pytest.fixture(scope="module")
def product_phase(tmp_path_factory):
    """For every product of a CTA: its barrier and the parity that is waited for."""
    where = tmp_path_factory.mktemp("phases")
    (where / "phases.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(where / "phases.cpp"), "-o", str(where / "phases")], check=True)
    out = subprocess.run([str(where / "phases")], check=True, capture_output=True, text=True).stdout
    return [tuple(int(x) for x in line.split()) for line in out.splitlines()]


def build(items, rescales, product_phase):
    """One CTA on items of so many key tiles; rescales[w]: in which tiles softmax warp w rescales O."""
    g = Graph(lambda bar: 1)
    done = lambda bar, n: ("done", bar, n)  # noqa: E731
    total = sum(items)
    # the n-th product on its barrier completes phase n of it
    count, phase = {}, []
    for n in range(total):
        bar, parity = product_phase[n]
        phase.append((("Product", bar), count.get(bar, 0)))
        assert parity == phase[n][1] & 1
        count[bar] = count.get(bar, 0) + 1
    tile = lambda kind, n: ((kind, n & 1), n >> 1)  # barriers for even and odd tiles  # noqa: E731

    for operand, used in (("K", "KEmpty"), ("V", "VEmpty")):  # the producers
        last = None
        for n in range(total):
            if n >= 2:
                last = g.wait(*tile(used, n - 2), operand, last)
            last = g.event(("set", *tile(operand + "Full", n)), last)
            g.event(done(*tile(operand + "Full", n)), last)
    last = None
    for n, _ in enumerate(items):
        if n >= 2:
            last = g.wait(*tile("QEmpty", n - 2), "Q", last)
        last = g.event(("set", *tile("QFull", n)), last)
        g.event(done(*tile("QFull", n)), last)

    last, n = None, 0
    for i, tiles in enumerate(items):  # S = Q K^T
        last = g.wait(*tile("QFull", i), "S", last)
        for j in range(tiles):
            last = g.wait(*tile("KFull", n), "S", last)
            if n >= 2:
                last = g.wait(*phase[n - 2], "S", last)
            last = g.event(("issue S", n), last)
            g.event(done(*tile("KEmpty", n)), last)
            g.event(done(*tile("SFull", n)), last)
            n += 1
        g.event(done(*tile("QEmpty", i)), last)
    last, ran, n = None, None, 0
    for i, tiles in enumerate(items):  # O += P V
        for j in range(tiles):
            last = g.wait(*tile("PFull", n), "PV", last)
            last = g.wait(*tile("VFull", n), "PV", last)
            if j == 0 and i > 0:
                last = g.wait("OFree", i - 1, "PV", last)
            ran = g.event(("product", n), last, ran)
            g.event(done(*tile("VEmpty", n)), ran)
            g.event(done(*phase[n]), ran)
            n += 1
    for w, pattern in enumerate(rescales):  # softmax warps
        last, n = None, 0
        for i, tiles in enumerate(items):
            for j in range(tiles):
                last = g.wait(*tile("SFull", n), f"softmax {w}", last)
                if j > 0 and pattern(n):
                    last = g.wait(*phase[n - 1], f"softmax {w} (rescale)", last)
                last = g.event(("weights", w, n), last)
                g.event(done(*tile("PFull", n)), last)
                n += 1
            last = g.wait(*phase[n - 1], f"softmax {w} (end)", last)
            last = g.event(("output", w, i), last)
            g.event(done("OFree", i), last)
    return g, phase


PATTERNS = {"never": lambda n: False, "always": lambda n: True, "first": lambda n: n % 5 == 1, "odd": lambda n: n % 2 == 1}


@pytest.mark.parametrize("items", [[1], [2], [3], [9], [1, 1, 1, 1], [3, 1, 2], [2, 2, 2, 2], [7, 4, 1, 1, 5]], ids=str)
def test_every_wait_for_a_product_is_sound(items, product_phase):
    for a, b in itertools.combinations_with_replacement(PATTERNS.values(), 2):
        g, phase = build(items, (a, b), product_phase)
        anc = g.ancestors()
        assert g.faults(anc) == []
        # O is read when all of an item's products are complete
        for i in range(len(items)):
            for n in range(sum(items[: i + 1])):
                assert ("product", n) in anc["output", 0, i]


def test_one_barrier_for_all_products_would_not_do():
    """An item's end would be taken for reached while the product before its last is still to come."""
    one = [(0, n & 1) for n in range(64)]
    g, _ = build([3], (PATTERNS["never"],), one)
    assert any("may seem over to softmax 0 (end)" in f for f in g.faults(g.ancestors()))
