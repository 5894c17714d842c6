"""CPU: which operands of a call share memory (rnn_overlap.h), compiled for the
host, against sets of their words."""
import ctypes as C
import os
import random
import subprocess

import pytest

from conftest import ROOT

SOURCE = """
#include "rnn_overlap.h"
extern "C" int overlap(uint64_t pa, size_t na, size_t sa, size_t wa, uint64_t pb, size_t nb, size_t sb,
                       size_t wb) {
    return rnn_overlap({(const void *)pa, na, sa, wa}, {(const void *)pb, nb, sb, wb});
}
extern "C" int any(const uint64_t *p, const size_t *w) {
    const RnnRows out[2] = {rnn_block((const void *)p[0], w[0]), rnn_block((const void *)p[1], w[1])},
                  in[2] = {rnn_block((const void *)p[2], w[2]), rnn_block((const void *)p[3], w[3])};
    return rnn_any_overlap(out, in);
}
"""


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    src, so = d / "overlap.cpp", d / "overlap.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "rustnn_amd", "csrc"), str(src), "-o", str(so)], check=True)
    f = C.CDLL(str(so))
    f.overlap.argtypes = [C.c_uint64, C.c_size_t, C.c_size_t, C.c_size_t] * 2
    return f


def words(p, n, stride, w):
    return {p // 4 + r * stride + i for r in range(n) for i in range(w)} if p else set()


def test_against_sets(built):
    rng, seen = random.Random(1), [0, 0]
    for k in range(20000):
        rows = []
        for _ in range(2):
            w = rng.randint(0, 6)
            rows.append([4 * rng.randint(200, 260), rng.randint(0, 6), max(w, 1) + rng.randint(0, 9), w])
        if k % 2:
            rows[1][2] = rows[0][2] = max(rows[0][2], rows[1][2])  # columns of one buffer
        if k % 50 == 0:
            rows[0][0] = 0
        want = bool(words(*rows[0]) & words(*rows[1]))
        assert built.overlap(*rows[0], *rows[1]) == want, rows
        seen[want] += 1
    assert min(seen) > 4000


@pytest.mark.parametrize("at,want", [((0, 40, 80, 120), 0), ((0, 20, 80, 120), 1),
                                     ((0, 40, 36, 120), 1), ((0, 120, 80, 130), 1),
                                     ((0, 40, 80, 82), 0)])
def test_results_and_operands(built, at, want):
    p = (C.c_uint64 * 4)(*[4096 + 4 * v for v in at])
    assert built.any(p, (C.c_size_t * 4)(*[40, 30, 20, 10])) == want
