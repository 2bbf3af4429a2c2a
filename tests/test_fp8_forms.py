"""The form that a product with an epilogue takes (zunzuncito_amd/csrc/zz_fp8_form.h, built here for the
host): rules on sizes."""
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def both(tmp_path_factory):
    """both(cases): each one's kernel, and whether a launch holds it; a case is (packed rows, columns, rows, matrices, table, 8-bit)."""
    exe = tmp_path_factory.mktemp("form") / "fp8_form"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "fp8_form.cpp"), "-o", str(exe)], check=True)

    def run(cases):
        text = "\n".join(" ".join(str(int(v)) for v in c) for c in cases)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(cases)
        return [tuple(int(v) for v in line.split()) for line in out]
    return run


@pytest.fixture(scope="module")
def forms(both):
    return lambda cases: [v for v, _ in both(cases)]


def test_one_matrix(forms):
    """One row, some, hundreds and thousands; a matrix past the caches."""
    assert forms([(2816, 2112, 1, 1, 0, 0), (4096, 2816, 8192, 1, 0, 0), (4096, 2816, 8192, 1, 0, 1), (65600, 1088, 3, 1, 0, 0),
                  (65600, 1088, 20, 1, 0, 0), (65600, 1088, 20, 1, 0, 1)]) == [1, 9, 13, 15, 16, 16]


def test_8bit_tiles_are_asked_for(forms):
    sizes = [(o, i, p, e, t) for o in (33, 700, 2816, 5632, 40000) for i in (100, 700, 2816) for e, t in ((1, 0), (8, 1), (128, 1))
             for p in (1, 7, 60, 300, 2000, 30000)]
    assert all(v <= 9 or v >= 14 for v in forms([(*s, 0) for s in sizes]))
    assert {11, 12, 13} <= set(forms([(*s, 1) for s in sizes]))


def test_tables(forms):
    """1 to 32 rows an expert, spread by no rule that is known: small tiles, not those of 64 x 128, which
    took 1.6 times as long over even and skewed spreads; many rows: large ones."""
    for o, i, e in ((1408, 2816, 128), (2816, 704, 128), (3584, 2048, 32), (1536, 2048, 256), (4096, 1024, 128)):
        assert {v % 13 for v in forms([(o, i, e * per, e, 1, 0) for per in (1, 2)])} == {1}
        assert set(forms([(o, i, e * per, e, 1, 0) for per in (3, 5, 8, 17, 32)])) == {3}
        assert set(forms([(o, i, e * 512, e, 1, 0)])) <= {7, 9}
        assert set(forms([(o, i, e * per, e, 1, 1) for per in (8, 17, 32)])) == {12}


def test_small_tables(forms):
    """Up to 1024 workgroups of the few-row form a table takes what one matrix of its rows does."""
    for o, i, e, per in ((512, 512, 64, 9), (200, 300, 40, 30), (4096, 1024, 8, 20)):
        assert forms([(o, i, e * per, e, 1, 0)])[0] in (0, 1, 2, 14)


def test_most_tiles(both):
    """2^24 tiles of 128 x 128 are 2^32 threads, which no launch holds."""
    fits = lambda *c: both([(*c, 0)])[0][1]  # noqa: E731
    assert fits(2 * 8064, 5, 1 << 24, 1, 1) and fits(2 * 8128, 5, (1 << 24) - 1024, 1, 1)
    assert not fits(2 * 8191, 5, 1 << 24, 1, 1) and not fits(2 * 8191, 5, 1 << 24, 512, 1)
    assert fits(1 << 24, 128, 120, 120, 1) and not fits(1 << 24, 128, 300, 127, 1)


def some_sizes(table, eight, n=100000):
    """(packed rows, columns, rows, matrices, table, 8-bit) over the sizes that calls have"""
    rng = random.Random(2)
    size = lambda top: round(2 ** rng.uniform(0, top))  # noqa: E731
    return [(size(17), size(13), size(14), size(9) if table else 1, table, eight) for _ in range(n)]


def sizes_of(test, *names):
    """What a test is parametrised with, as dicts."""
    for mark in test.pytestmark:
        if mark.name == "parametrize":
            args = [a.strip() for a in mark.args[0].split(",")]
            if set(names) <= set(args):
                yield from (dict(zip(args, v)) for v in mark.args[1])


@pytest.mark.parametrize("gated", [False, True])
def test_exact_sums_are_tested_in_every_form(forms, gated):
    """The sizes of test_gpu_fp8_sums.py, which are run in both types, take every form there is."""
    import test_gpu_fp8_sums as T
    G = 2 if gated else 1
    for table, sizes in ((0, [(G * o, i, s, 1, 0, 0) for s, o, i in T.SINGLE]), (1, [(G * o, i, p, e, 1, 0) for e, p, o, i in T.TABLES])):
        assert set(forms(sizes)) == set(forms(some_sizes(table, 0)))


@pytest.mark.parametrize("gated", [False, True])
def test_8bit_tiles_are_tested_in_every_form(forms, gated):
    """test_gpu_fp8_eight.py has each of the three 8-bit tiles, for one matrix and for tables, plain and
    gated."""
    import test_gpu_fp8_eight as T
    G = 2 if gated else 1
    one, table = [], []
    for f in (v for k, v in vars(T).items() if k.startswith("test_")):
        mine = [d for d in sizes_of(f, "O", "I") if d.get("gated", gated) == gated]
        one += [(G * d["O"], d["I"], d["S"], 1, 0, 1) for d in mine if "S" in d]
        table += [(G * d["O"], d["I"], d["P"], d["E"], 1, 1) for d in mine if "P" in d]
    for t, sizes in ((0, one), (1, table)):
        assert {11, 12, 13} <= set(forms(sizes))
        assert {11, 12, 13} == {v for v in forms(some_sizes(t, 1)) if 10 < v < 14}
