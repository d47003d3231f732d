"""The epilogue's walk over its accumulators when a wait runs out, with the
barriers played on the host."""
import os
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "ark_ring.h"

// A barrier as mbarrier.try_wait.parity sees it: the phase of the given parity has
// completed if the one that is under way has the other parity.  It completes `last`
// phases and no more.
struct Barrier {
    unsigned done = 0, last;
    bool passed(unsigned parity) const { return (done & 1) != parity; }
};

int main(int, char** argv) {
    const unsigned items = atoi(argv[1]);
    Barrier b[2];
    b[0].last = atoi(argv[2]), b[1].last = atoi(argv[3]);
    ark::Ring<2> r;
    ark::until_lost(0, items, 1, [&](unsigned) {
        // the writer completes the next phase as soon as the reader waits, until it stops
        Barrier& x = b[r.at];
        if (!x.passed(r.parity) && x.done < x.last) ++x.done;
        if (!x.passed(r.parity)) return false;
        putchar('1');
        r.next();
        return true;
    }, [&](unsigned) { putchar('0'); });
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "ark_b200", "csrc"), str(d / "ring.cpp"),
                    "-o", str(d / "ring")], check=True)
    return str(d / "ring")


@pytest.mark.parametrize("first,second", [(0, 0), (1, 0), (1, 1), (2, 1), (2, 2), (3, 2), (9, 9)])
def test_nothing_is_ready_after_a_wait_that_ran_out(program, first, second):
    """Item i uses buffer i % 2: the items whose phases completed, and none behind them."""
    items = 12
    out = subprocess.run([program, str(items), str(first), str(second)], capture_output=True, text=True, check=True)
    ready = min(items, first + second)
    assert out.stdout == "1" * ready + "0" * (items - ready)
