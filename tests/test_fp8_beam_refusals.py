"""What the 8-bit rows, the fp8 product and the beam calls decline, and that they say why. The
arguments are looked at before anything else, so these run without a device; where there is
one, only pointers that no check lets through are passed."""
import ctypes as C
import subprocess
import os

import numpy as np
import pytest

import zunzuncito_amd as zz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20                      # pretended device addresses, far apart
X, R, S_, Q, SC, W = (A * (i + 1) * 64 for i in range(6))


def test_headers_compile_as_c():
    src = '#include "zz_fp8.h"\n#include "zz_beam.h"\nint main(void){ return ZZ_BF16 + ZZ_BEAM_MAXW; }\n'
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"),
                        "-x", "c", "-"], input=src, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_sizes():
    assert [zz.fp8_row_bytes(d) for d in (1, 128, 129, 2816, 1088)] == [128, 128, 256, 2816, 1152]
    assert zz.lib().zz_fp8_row_bytes(0) == -1
    assert zz.beam_ws_bytes(1, 1, 1) > 0
    for n, w, v in ((0, 1, 1), (1, 0, 1), (1, 17, 9), (1, 1, 0), (1, 1, zz.ZZ_BEAM_MAXV + 1), (1 << 16, 1, 1), (1 << 15, 2, 1)):
        assert zz.lib().zz_beam_ws_bytes(n, w, v) == -1
        with pytest.raises(RuntimeError):
            zz.beam_ws_bytes(n, w, v)
    assert zz.beam_ws_bytes(16, 8, 262144) <= 16 * 8 * (262144 // 8 + 65536)


NORM = dict(d_x=X, d_res=R, d_sum=S_, d_w=W, S=4, D=256, eps=1e-6, d_q=Q, d_s=SC)


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(d_x=0), "bad arguments"), (dict(d_q=0), "bad arguments"),
    (dict(d_s=0), "bad arguments"), (dict(S=0), "bad arguments"), (dict(S=-1), "bad arguments"),
    (dict(S=(1 << 20) + 1), "bad arguments"), (dict(D=0), "bad arguments"), (dict(D=8193), "8192"),
    (dict(ldx=255), "closer"), (dict(ldr=255), "closer"), (dict(lds=255), "closer"), (dict(ldx=-256), "closer"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(d_x=X + 2), "misaligned"), (dict(d_res=R + 1), "misaligned"), (dict(d_sum=S_ + 2), "misaligned"),
    (dict(d_w=W + 2), "misaligned"), (dict(d_q=Q + 8), "misaligned"), (dict(d_s=SC + 2), "misaligned"),
    (dict(d_x=X + 1, dtype=1), "misaligned"),
    (dict(d_sum=X, ldx=512), "overlaps"),            # the same buffer, rows elsewhere
    (dict(d_sum=X + 16), "overlaps"), (dict(d_sum=R + 16), "overlaps"), (dict(d_q=X + 64), "overlaps"),
    (dict(d_s=Q), "overlaps"), (dict(d_s=S_), "overlaps"), (dict(d_w=S_), "overlaps"), (dict(d_w=Q + 16), "overlaps"),
])
def test_add_norm_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.add_norm_fp8_dev(**{**NORM, **bad})


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=7), "dtype"), (dict(d_x=0), "bad arguments"), (dict(S=0), "bad arguments"), (dict(D=0), "bad arguments"),
    (dict(D=(1 << 20) + 1), "2\\^20"), (dict(S=1 << 20, D=128 * 129), "2\\^27"), (dict(ldx=100), "closer"),
    (dict(d_x=X + 2), "misaligned"), (dict(d_q=X), "overlaps"), (dict(d_s=Q + 16), "overlaps"),
])
def test_rows_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.rows_fp8_dev(**{**dict(d_x=X, S=4, D=256, d_q=Q, d_s=SC), **bad})


def test_matrix_declines():
    for O, I in ((0, 8), (8, 0), (-1, 8), ((1 << 24) + 1, 8), (8, (1 << 16) + 1), (1 << 20, 1 << 15)):
        with pytest.raises(RuntimeError, match="bad shape"):
            zz.Fp8Matrix(O, I)
    L = zz.lib()

    def mm(mat=-1, q=Q, s=SC, S=4, dtype=0, y=X, ldy=0):
        assert L.zz_fp8_matmul_dev(mat, q, s, S, dtype, y, ldy, None) == 0
        return zz.last_error()

    assert "dtype" in mm(dtype=3)
    for kw in (dict(q=None), dict(s=None), dict(y=None), dict(S=0), dict(S=(1 << 20) + 1), dict(ldy=-1)):
        assert "bad arguments" in mm(**kw)
    for kw in (dict(q=Q + 4), dict(s=SC + 1), dict(y=X + 2), dict(y=X + 1, dtype=1)):
        assert "misaligned" in mm(**kw)
    assert "gpu_init" in mm() or "no such matrix" in mm()
    y = np.full((1, 4), 7.0, np.float32)
    x = np.ones((1, 4), np.float32)
    assert L.zz_fp8_matmul(-1, x.ctypes.data_as(zz._f32p), y.ctypes.data_as(zz._f32p), 1) == 0
    assert L.zz_fp8_matmul(-1, x.ctypes.data_as(zz._f32p), y.ctypes.data_as(zz._f32p), 0) == 0
    assert "bad arguments" in zz.last_error() and np.all(y == 7.0)
    assert L.zz_fp8_upload(-1, None, None) == 0 and L.zz_fp8_upload_dev(-1, Q, SC + 2) == 0
    L.zz_fp8_destroy(-1)                             # nothing to give back
    L.zz_fp8_destroy(1 << 20)


STEP = dict(d_logits=X, N=2, W=3, V=1000, d_score=R, d_score_out=S_, d_parent=Q, d_token=SC, d_ws=W, ws_bytes=1 << 20,
            d_done=A, d_done_out=2 * A)


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=2), "dtype"), (dict(N=0), "W <="), (dict(W=0), "W <="), (dict(W=17), "W <="), (dict(V=0), "V <="),
    (dict(V=zz.ZZ_BEAM_MAXV + 1), "V <="), (dict(N=65535, W=2), "65535"),
    (dict(d_logits=0), "bad arguments"), (dict(d_score=0), "bad arguments"), (dict(d_score_out=0), "bad arguments"),
    (dict(d_parent=0), "bad arguments"), (dict(d_token=0), "bad arguments"), (dict(d_ws=0), "bad arguments"),
    (dict(ldl=999), "bad arguments"), (dict(d_logits=X + 2), "misaligned"), (dict(d_logits=X + 1, dtype=1), "misaligned"),
    (dict(d_score=R + 1), "misaligned"), (dict(d_parent=Q + 2), "misaligned"), (dict(d_ws=W + 4), "misaligned"),
    (dict(ws_bytes=100), "workspace"), (dict(d_parent=R), "overlaps"), (dict(d_score_out=R + 4), "overlaps"),
    (dict(d_ws=X + 8), "overlaps"), (dict(d_token=Q + 4), "two outputs"), (dict(d_ws=S_ - 8), "two outputs"),
    (dict(d_done_out=A + 1), "overlaps"),
])
def test_step_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.beam_step_dev(**{**STEP, **bad})


ORD = dict(d_dst=X, d_src=R, d_parent=Q, N=2, W=3, outer=2, outer_stride=6000, row_stride=1000, row_bytes=900)


@pytest.mark.parametrize("bad, why", [
    (dict(d_dst=0), "bad arguments"), (dict(d_src=0), "bad arguments"), (dict(d_parent=0), "bad arguments"),
    (dict(d_parent=Q + 2), "bad arguments"), (dict(N=0), "bad arguments"), (dict(W=0), "bad arguments"),
    (dict(W=17), "bad arguments"), (dict(outer=0), "bad arguments"), (dict(row_bytes=0), "bad arguments"),
    (dict(row_bytes=1001), "bad arguments"), (dict(outer_stride=5999), "planes overlap"),
    (dict(row_stride=-1000), "bad arguments"), (dict(d_dst=R + 4), "overlaps src"), (dict(d_dst=Q - 100), "overlaps parent"),
])
def test_reorder_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.beam_reorder_dev(**{**ORD, **bad})


def test_stack_beam_declines():
    L = zz.lib()
    assert L.zz_stack_beam_dev(-1, X, 4, 2, -1, R, Q, None) == 0
    assert "zz_stack_beam_dev" in zz.last_error()


@pytest.mark.parametrize("bad, why", [
    (dict(tok=None), "bad arguments"), (dict(seq=None), "bad arguments"), (dict(score=None), "bad arguments"),
    (dict(W=0), "bad arguments"), (dict(W=17), "bad arguments"), (dict(n=-1), "bad arguments"),
    (dict(n=(1 << 24) + 1), "bad arguments"), (dict(tok=X + 2), "misaligned"), (dict(seq=R + 1), "misaligned"),
    (dict(score=Q + 2), "misaligned"), (dict(tok=R + 40), "overlaps"), (dict(score=R + 44), "overlaps"),
    (dict(tok=Q + 12), "overlaps"),
])
def test_stack_beam_arguments(bad, why):
    """The arguments are looked at before the stack, and before anything is written."""
    a = {**dict(tok=X, W=4, n=2, eos=-1, seq=R, score=Q), **bad}
    assert zz.lib().zz_stack_beam_dev(-1, a["tok"], a["W"], a["n"], a["eos"], a["seq"], a["score"], None) == 0
    assert why in zz.last_error()
