"""Whether strided views share bytes (csrc/overlap.hpp), against sets of addresses; and the calls that refuse such views."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from pequegrad_b200 import _lib as L
from test_generation_cpu import CACHE, INT8, attend, logits, read, refused, t, write

CSRC = Path(L.__file__).parent / "csrc"

SHIM = """
#include "overlap.hpp"
using namespace pgb;
static ByteView make(const int64_t *v) {
  ByteView b((uintptr_t)v[0], v[1]);
  for (int i = 0; i < v[2]; ++i) b.add(v[3 + 2 * i], v[4 + 2 * i]);
  return b;
}
extern "C" int share(const int64_t *a, const int64_t *b) { return views_share(make(a), make(b)); }
extern "C" int itself(const int64_t *a) { return view_overlaps_itself(make(a)); }
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-Wall", "-Werror", f"-I{CSRC}", str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    return C.CDLL(str(d / "shim.so"))


def flat(base, length, dims):
    v = [base, length, len(dims)]
    for n, s in dims:
        v += [n, s]
    return (C.c_int64 * len(v))(*v)


def starts(base, dims):
    out = [base]
    for n, s in dims:
        out = [a + i * s for a in out for i in range(n)]
    return out


def some_view(rng):
    dims = [(rng.choice([1, 1, 2, 3, 5]), rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 40, 48])) for _ in range(rng.randint(0, 4))]
    return rng.randint(100, 160), rng.choice([1, 2, 4, 8]), dims


def test_against_sets_of_addresses(shim):
    rng = random.Random(3)
    met = [0, 0, 0, 0]
    for _ in range(30000):
        a, b = some_view(rng), some_view(rng)
        if rng.random() < 0.5:
            b = (b[0], a[1], a[2])  # the same layout somewhere else, as the parts of a packed buffer have
        bytes_of = [[x + i for x in starts(v[0], v[2]) for i in range(v[1])] for v in (a, b)]
        twice = len(set(bytes_of[0])) < len(bytes_of[0])
        common = bool(set(bytes_of[0]) & set(bytes_of[1]))
        assert shim.itself(flat(*a)) == twice, a
        assert shim.share(flat(*a), flat(*b)) == common, (a, b)
        met[twice] += 1
        met[2 + common] += 1
    assert min(met) > 2000


def test_views_as_large_as_a_gpu(shim):
    # the layouts that calls have, 2^36 bytes and more: pages of K and V in turn, heads inside and outside of the slots
    pages, heads, slots, D = 1 << 20, 8, 64, 256
    row, page = D, heads * slots * D
    for order in ([(pages, 2 * page), (heads, slots * row), (slots, row)], [(pages, 2 * page), (heads, row), (slots, heads * row)]):
        a, b = flat(1 << 40, D, order), flat((1 << 40) + page, D, order)
        assert not shim.itself(a) and not shim.share(a, b) and shim.share(a, flat((1 << 40) + page - 16, D, order))
        # a page that holds its scales behind its values
        packed = [(pages, page + heads * slots * 4), *order[1:]]
        scales = flat((1 << 40) + page, slots * 4, [(pages, page + heads * slots * 4), (heads, slots * 4)])
        assert not shim.share(flat(1 << 40, D, packed), scales)
        assert shim.share(flat(1 << 40, D, packed), flat((1 << 40) + page - 16, slots * 4, [(pages, page + heads * slots * 4)]))
        assert shim.itself(flat(1 << 40, D, [(pages, page - 16), *order[1:]]))
    # no rows at all share nothing
    assert not shim.share(flat(0, 64, [(0, 64)]), flat(0, 64, [(5, 64)])) and not shim.itself(flat(0, 64, [(0, 0)]))


def test_written_views_whose_pitches_overlap_together_are_refused():
    """Each pitch is long enough for a row by itself; all of them are the same."""
    bad = L.ERR_INVALID_ARG
    refused(read(k=t((5, 4, 64), strides=(64, 64, 1))), bad, b"k overlaps itself")
    refused(read(v=t((5, 4, 64), strides=(128, 64, 1))), bad, b"v overlaps itself")
    refused(attend(out=t((5, 8, 64), strides=(64, 64, 1))), bad, b"out overlaps itself")
    refused(write(kc=t(CACHE, strides=(2048, 64, 64, 1))), bad, b"k_cache overlaps itself")
    refused(write(vc=t(CACHE, strides=(4 * 2048 - 64, 2048, 64, 1))), bad, b"v_cache overlaps itself")
    refused(write(**{**INT8, "ks": t(CACHE[:3], L.F32, strides=(32, 32, 1))}), bad, b"the scales overlap themselves")
    refused(logits(out=t((3, 100), strides=(99, 1))), bad, b"out overlaps itself")
