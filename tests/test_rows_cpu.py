"""The host's arithmetic on strided rows (csrc/rows.cuh) against sets of bytes."""
import ctypes
import pathlib
import random
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).parents[1] / "halftone_quantizedkvcache_b200" / "csrc"
SHIM = """
#include "rows.cuh"
static hq::Rows of(const long long* a) {
  return hq::rows_of(reinterpret_cast<const void*>(a[0]), a[1], a[2], a[3], a[4], a[5]);
}
extern "C" int meet(const long long* a, const long long* b) { return hq::rows_meet(of(a), of(b)); }
extern "C" int meet_each_other(const long long* a) { return hq::rows_meet(of(a)); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("rows")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), str(d / "shim.cpp"), "-o", str(d / "shim.so")],
                   check=True)
    return ctypes.CDLL(str(d / "shim.so"))


def rows(base, n0, n1, s0, s1, size):
    return [range(base + i * s0 + h * s1, base + i * s0 + h * s1 + size) for i in range(n0) for h in range(n1)]


def args(r):
    return (ctypes.c_longlong * 6)(*r)


def test_against_sets_of_bytes(lib):
    rng = random.Random(7)
    both = [0, 0]
    for _ in range(20000):
        size = rng.choice([1, 4, 16])
        s = [rng.choice([rng.randint(-120, 120), size * rng.randint(-8, 8), 4 * size, 0]) for _ in range(4)]
        if rng.random() < 0.6:
            s[2] = s[0]
        if rng.random() < 0.6:
            s[3] = s[1]
        a = (5000 + rng.randint(0, 60), rng.randint(1, 6), rng.randint(1, 5), s[0], s[1], size)
        b = (5000 + rng.randint(-200, 400), rng.randint(1, 6), rng.randint(1, 5), s[2], s[3], rng.choice([size, 2 * size]))
        ra, rb = rows(*a), rows(*b)
        want = not set().union(*ra).isdisjoint(set().union(*rb))
        assert lib.meet(args(a), args(b)) == want == lib.meet(args(b), args(a)), (a, b)
        want_self = len(set().union(*ra)) < sum(map(len, ra))
        assert lib.meet_each_other(args(a)) == want_self, a
        both[want] += 1
    assert min(both) > 3000


def test_layouts_as_callers_have_them(lib):
    # q, k and v in one projection's rows; K and V halves of one array; rows apart, one row into the other
    w = 2 * 32 * 128
    q, k, v = (10 ** 12, 5000, 16, w, 256, 256), (10 ** 12 + 16 * 256, 5000, 8, w, 256, 256), (10 ** 12 + 24 * 256, 5000, 8, w, 256, 256)
    for a, b in ((q, k), (k, v), (q, v)):
        assert not lib.meet(args(a), args(b))
    for a in (q, k, v):
        assert lib.meet(args(a), args(a)) and not lib.meet_each_other(args(a))
    assert lib.meet(args(q), args((k[0] - 256, *k[1:])))
    assert lib.meet(args(k), args((k[0] + w, *k[1:])))
    assert not lib.meet(args(k), args((k[0] + 5000 * w, *k[1:])))
    assert lib.meet_each_other(args((10 ** 12, 5000, 8, 256, 256, 256)))
    assert lib.meet(args((10 ** 12, 1 << 20, 8, 2048, 256, 256)), args((10 ** 12 + 5, 3, 1, 7, 0, 1)))
