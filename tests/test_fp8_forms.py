"""The form that a product with an epilogue takes (zunzuncito_amd/csrc/zz_fp8_form.h, built here for the
host): rules on sizes."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    """forms(cases): each one's kernel; a case is (packed rows, columns, rows, matrices, table, 8-bit)."""
    exe = tmp_path_factory.mktemp("form") / "fp8_form"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "fp8_form.cpp"), "-o", str(exe)], check=True)

    def run(cases):
        text = "\n".join(" ".join(str(int(v)) for v in c) for c in cases)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split()
        assert len(out) == len(cases)
        return [int(v) for v in out]
    return run


def test_one_matrix(forms):
    """One row, some, hundreds and thousands; a matrix past the caches."""
    assert forms([(2816, 2112, 1, 1, 0, 0), (4096, 2816, 8192, 1, 0, 0), (4096, 2816, 8192, 1, 0, 1), (65600, 1088, 3, 1, 0, 0),
                  (65600, 1088, 20, 1, 0, 0), (65600, 1088, 20, 1, 0, 1)]) == [1, 9, 13, 15, 16, 16]


def test_8bit_tiles_are_asked_for(forms):
    sizes = [(o, i, p, e, t) for o in (33, 700, 2816, 5632, 40000) for i in (100, 700, 2816) for e, t in ((1, 0), (8, 1), (128, 1))
             for p in (1, 7, 60, 300, 2000, 30000)]
    assert all(v <= 9 or v >= 14 for v in forms([(*s, 0) for s in sizes]))
    assert {11, 12, 13} <= set(forms([(*s, 1) for s in sizes]))
