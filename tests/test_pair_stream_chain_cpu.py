"""Kernels that start before the kernel ahead of them has ended read what it writes by coherent loads: a check of the source,
because a stale or early read depends on timing and need not show in a result."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "fold_cp_ops_b200" / "csrc"
NON_COHERENT = re.compile(r"__ldg\s*\(|ld\.global\.nc|__restrict__")


def functions(text):
    """``name -> body`` of the functions that begin in the first column of a source file."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    text = re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text)
    out, at = {}, 0
    while (m := re.compile(r"^[a-zA-Z_][^;{}#]*?\b(\w+)\s*\([^;{}]*\)\s*\{", re.M).search(text, at)) is not None:
        depth, end = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        out[m.group(1)] = text[m.start():end]
        at = end
    return out


def reaches(bodies, name, seen=()):
    """The function and the file's functions that it calls."""
    names = {name, *seen}
    for other in bodies:
        if other not in names and re.search(rf"\b{other}\b", bodies[name]):
            names |= reaches(bodies, other, tuple(names))
    return names


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("pair_*.cu")))
def test_kernels_of_a_chain_read_no_predecessors_data_through_the_read_only_path(source):
    bodies = functions((CSRC / source).read_text())
    kernels = [n for n, b in bodies.items() if "__global__" in b.split("(")[0]]
    assert len(kernels) == (CSRC / source).read_text().count("__global__")
    for kernel in kernels:
        if "behind_previous()" not in bodies[kernel]:
            continue
        for name in reaches(bodies, kernel):
            assert not NON_COHERENT.search(bodies[name]), f"{source}: {kernel} runs behind another kernel, but {name} reads past the caches' order"


def test_every_early_kernel_waits():
    """A kernel that is launched to start early begins with the wait, before it reads memory."""
    for source in sorted(CSRC.glob("pair_*.cu")):
        text = source.read_text()
        bodies = functions(text)
        for name in set(re.findall(r"launch_behind\(\s*(\w+)", text)) & set(bodies):
            head = re.split(r"\bbehind_previous\(\);", bodies[name])
            assert len(head) == 2 and "[" not in head[0].split("{", 1)[1], f"{source.name}: {name}"
