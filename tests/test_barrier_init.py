"""fence.mbarrier_init covers the initialisations of the thread that executes it: whoever initialises barriers fences them itself, under the same condition."""
import glob
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pegainfer_b200", "csrc")
SOURCES = sorted(p for p in glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) if "mbar_init(" in open(p).read() and not p.endswith("common.cuh"))


def guards(lines, at):
    """line numbers of the conditions that the statement in line `at` stands under, innermost first: blocks by their braces, single statements by their indentation"""
    out, depth = [], len(lines[at]) - len(lines[at].lstrip())
    if lines[at].lstrip().startswith("if ("):
        out.append(at)
    for i in range(at - 1, -1, -1):
        text = lines[i].strip()
        if not text or text.startswith(("#", "//")):
            continue
        here = len(lines[i]) - len(lines[i].lstrip())
        if here < depth:
            depth = here
            if text.startswith("if ("):
                out.append(i)
        if here == 0:
            break
    return out


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_every_thread_fences_the_barriers_that_it_initialises(path):
    lines = open(path).read().split("\n")
    fences = [i for i, x in enumerate(lines) if "mbar_fence_init();" in x]
    for i, x in enumerate(lines):
        if "mbar_init(" not in x:
            continue
        behind = [f for f in fences if f > i]
        assert behind, (path, i + 1)
        assert guards(lines, i)[:1] == guards(lines, behind[0])[:1], f"{os.path.basename(path)}:{i + 1} and the fence in line {behind[0] + 1}"
