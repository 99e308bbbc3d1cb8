"""The search of a draw's border (top_k, top_p) on the host: the same source that the kernels run, by one lane.

A border is right if its entry reaches the aim and the entries before it do not, both within what sums of 64-bit weights may be
off: n terms of one sign, each addition half a step of 2^-52, n 2^-53 of the sum, and twice that for sums in two orders.  The
smallest weights are 2^-1074, so 1e-320 is added for what lies below every number."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOG2E = 1.4426950408889634
FORMS = {"block": 0, "wave": 1, "four lanes": 2, "short list": 3}


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("border") / "border_search.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-fPIC", "-shared", "-I",
                           os.path.join(ROOT, "isaaclab_amd", "csrc"), os.path.join(ROOT, "tests", "workers", "border_search.cpp"),
                           "-o", so])
    fn = C.CDLL(so).border_search
    fn.restype = C.c_long
    fn.argtypes = [C.c_int, C.c_void_p, C.c_void_p, C.c_long, C.c_double, C.c_double, C.c_int, C.c_double, C.c_long, C.c_void_p, C.c_void_p]

    def call(form, x, w=None, c=LOG2E, p=1.0, k=0, aim=0.0, most=64):
        x, tau, place = np.ascontiguousarray(x, np.float32), C.c_float(), C.c_int()
        w = None if w is None else np.ascontiguousarray(w, np.float64)
        n = fn(FORMS[form], x.ctypes.data, None if w is None else w.ctypes.data, len(x), c, float(np.float32(p)), k, aim, most,
               C.byref(tau), C.byref(place))
        assert n >= 0, f"more than {most} passes over the row"
        return n, tau.value, place.value

    return call


def check(x, w, aim, tau, place):
    x = np.asarray(x, np.float32)
    kept = (x > tau) | ((x == tau) & (np.arange(len(x)) <= place))
    assert kept.any(), (tau, place)
    tau = x[kept].min()
    place = np.flatnonzero(kept & (x == tau))[-1]
    before = np.sum(w[(x > tau) | ((x == tau) & (np.arange(len(x)) < place))])
    off = 2 * len(x) * 2.0 ** -53 * np.sum(w) + 1e-320
    assert before < aim + off and before + w[place] >= aim - off, (before, w[place], aim)


def weights(x, c=LOG2E):
    x = np.asarray(x, np.float64)
    return np.exp2((x - x.max()) * c)


@pytest.mark.parametrize("n, spread, form", [(n, s, f) for n, s in ((1000, 0.1), (4096, 2.0)) for f in FORMS] +
                         [(131072, 0.1, "block"), (131072, 0.1, "short list")])
def test_a_peak_and_a_tail(search, n, spread, form):
    """The tail weighs less than a unit of the fixed point an entry, and holds the border: a few passes, not one a bucket.

    A level takes a histogram, a look at the bucket, log2(buckets) more for a miss, and one to cut it: 6 + 3 or 12 + 3.  The first
    one misses; those behind it weigh in units of what is left and miss by a bucket at most, 4 passes each, of which 32 bits of keys
    take 6 by 62 buckets, 3 by 4094: 9 + 24 or 15 + 12."""
    g = np.random.default_rng(n)
    for peak in (2.0, 10.0, 15.0, 20.0, 22.8, 23.0, 24.0, 30.0, 36.0, 40.0):
        x = g.normal(0.0, spread, n).astype(np.float32)
        x[n // 3] = peak
        w = weights(x)
        for p in (0.5, 0.9, 0.9999, 0.99995, 0.99999, 1 - 2.0 ** -23):
            p = float(np.float32(p))
            _, tau, place = search(form, x, p=p, most=36)
            check(x, w, p * w.sum(), tau, place)


@pytest.mark.parametrize("form", FORMS)
def test_many_levels(search, form):
    """Peaks over peaks, each a share of 2^-k below the one before, rows in order, few values, values far apart."""
    g = np.random.default_rng(7)
    n = 3000
    rows = [np.concatenate([[-3.0 * j] * (j * j + 1) for j in range(20)]),
            np.linspace(0.0, -700.0, n), np.linspace(-40.0, 0.0, n), -np.abs(g.standard_cauchy(n)) * 5,
            np.round(g.normal(0, 1, n)), g.normal(0, 1, n) * 10.0 ** g.integers(-30, 3, n), np.full(n, -3.0),
            np.where(np.arange(n) % 3 == 0, -np.inf, g.normal(0, 4, n))]
    for x in rows:
        x = x.astype(np.float32)
        for c in (LOG2E, LOG2E / 0.05, LOG2E / 50.0):
            w = weights(x, c)
            for p in (0.0, 1e-6, 0.3, 0.77, 0.9999, 0.9999999):
                p = float(np.float32(p))
                _, tau, place = search(form, x, c=c, p=p)
                check(x, w, max(p * w.sum(), 1e-300), tau, place)
            for k in (1, 2, 61, 700):
                if k >= np.isfinite(x).sum():
                    continue
                _, tau, place = search(form, x, c=c, k=k)
                assert place == np.lexsort((np.arange(len(x)), -x))[k - 1] and x[place] == tau


@pytest.mark.parametrize("form", FORMS)
def test_an_aim_at_the_end_of_the_sums(search, form):
    """An aim that the row's weights reach in one order of addition and miss by their last bit in another: the border is an entry
    of the row all the same, one of those at which the sum ends."""
    short = 0
    for seed in range(400):                             # the end of the row
        g = np.random.default_rng(seed)
        n = int(g.integers(20, 300))
        x = g.normal(0, 2, n).astype(np.float32)
        w = weights(x)
        aim = float(max(np.sum(w), np.cumsum(w)[-1], np.cumsum(np.sort(w))[-1], np.cumsum(np.sort(w)[::-1])[-1]))
        short += aim > np.cumsum(w)[-1]
        _, tau, place = search(form, x, w, aim=aim)
        check(x, w, aim, tau, place)
    assert short > 20                                   # it happened
    for seed in range(400):                             # between two entries
        g = np.random.default_rng(seed)
        n = int(g.integers(20, 300))
        x = g.normal(0, 2, n).astype(np.float32) if seed % 2 else np.round(g.normal(0, 3, n)).astype(np.float32)
        w = weights(x, LOG2E / 3)
        first = np.sort(w)[::-1][:int(g.integers(1, n))]
        for aim in (np.sum(first), np.cumsum(first)[-1], np.cumsum(first[::-1])[-1], np.cumsum(first)[-1] * (1 + 2.0 ** -52)):
            _, tau, place = search(form, x, w, c=LOG2E / 3, aim=float(aim))
            check(x, w, float(aim), tau, place)
