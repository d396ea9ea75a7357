"""Kernels that start while the kernel in front still runs (pdl_wait): what they read behind the wait is not declared as data that nobody writes. The declaration
(const __restrict__, or a load through __ldg) lets the compiler move such a load in front of the wait, or take the path for constant data. CPU only: the sources are
looked at."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashrt_b200", "csrc")


def kernels(name):
    """(name, parameters, body) of every kernel of a source."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s+)?(\w+)\(", text):
        def close(at, pair):
            depth = 0
            for i in range(at, len(text)):
                depth += (text[i] == pair[0]) - (text[i] == pair[1])
                if depth == 0:
                    return i
        end = close(m.end() - 1, "()")
        start = text.index("{", end)
        yield m.group(1), text[m.end():end], text[start:close(start, "{}") + 1]


@pytest.mark.parametrize("source,least", [("frx_sort.cu", 7), ("frx_mxfp4.cu", 4)])
def test_loads_behind_the_wait_are_ordinary_ones(source, least):
    seen = 0
    for name, params, body in kernels(source):
        if "pdl_wait()" not in body:
            continue
        seen += 1
        assert not re.search(r"\bconst\b[^,]*\*\s*__restrict__", params), name
        assert "__ldg(" not in body, name
    assert seen >= least


def test_the_sources_are_read_as_meant():
    names = [k[0] for k in kernels("frx_sort.cu")]
    assert {"k_sort_count", "k_sort_scan", "k_sort_place", "k_rows_out", "k_rows_back", "k_rows_back_grad", "k_route_grad"} <= set(names)
