"""The bounds that the kernels joining the attention's partials put on a row's entry, which holds anything
when the attention gave up before it wrote it (compiled for the host; no GPU needed)."""
import ctypes
import itertools
import os
import random
import subprocess

import pytest

from conftest import PKG


@pytest.fixture(scope="module")
def partials_exist(tmp_path_factory):
    d = tmp_path_factory.mktemp("partials")
    src, so = d / "t.cpp", d / "t.so"
    src.write_text('#include "partials.h"\n'
                   'extern "C" int inside(int f, int c, int p) { return ds::partials_exist(f, c, p); }\n')
    subprocess.run(["g++", "-shared", "-fPIC", "-O2", "-fsanitize=signed-integer-overflow",
                    "-fsanitize-undefined-trap-on-error", "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(so)],
                   check=True, capture_output=True)
    return ctypes.CDLL(str(so)).inside


def test_entries_outside_the_workspace_are_rejected(partials_exist):
    top = 2 ** 31 - 1
    edges = [-top - 1, -top, -2, -1, 0, 1, 2, 31, 32, 33, 147, 148, 295, 296, 297, top - 296, top - 1, top]
    rng = random.Random(1)
    entries = list(itertools.product(edges, edges))
    entries += [(rng.randint(-top - 1, top), rng.randint(-top - 1, top)) for _ in range(2000)]
    entries += [(rng.randint(0, 300), rng.randint(0, 300)) for _ in range(2000)]
    for parts in (1, 2, 148, 296):
        for first, count in entries:
            # partials first .. first + count - 1 of 0 .. parts - 1
            want = first >= 0 and count >= 0 and first + count <= parts
            assert bool(partials_exist(first, count, parts)) == want, (first, count, parts)


def test_a_row_s_own_entries_are_accepted(partials_exist):
    for parts in (1, 7, 296):
        assert all(partials_exist(f, n, parts) for f in range(parts) for n in range(parts - f + 1))
