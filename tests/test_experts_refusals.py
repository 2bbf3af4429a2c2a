"""What the sorting by expert, the way back, its gradient, the product's epilogue and the tables of
experts decline, and that they say why. The arguments are looked at before anything else, so these
run without a device; where there is one, only pointers that no check lets through are passed."""
import os
import subprocess

import numpy as np
import pytest

import zunzuncito_amd as zz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 26                      # pretended device addresses, far apart
IDS, OFFS, ROW, POS, X, XS, WS, W, OUT, Q, SC, Y = (A * (i + 1) for i in range(12))
NAN, INF = float("nan"), float("inf")


def test_header_compiles_as_c():
    src = '#include "zz_experts.h"\nint main(void){ return ZZ_EP_SILU + ZZ_EXPERTS_MAXE; }\n'
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"),
                        "-x", "c", "-"], input=src, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_sizes():
    assert zz.experts_ws_bytes(1, 1, 1) > 0 and zz.experts_ws_bytes(1 << 20, 16, 512) <= 256 * 512 * 4
    for bad in ((0, 1, 1), ((1 << 20) + 1, 1, 1), (1, 0, 1), (1, 17, 32), (1, 1, 0), (1, 1, 513), (-1, 1, 1)):
        assert zz.lib().zz_experts_ws_bytes(*bad) == -1
        with pytest.raises(RuntimeError, match="declined"):
            zz.experts_ws_bytes(*bad)


DISPATCH = dict(d_eidx=IDS, S=300, K=4, E=16, d_offs=OFFS, d_row=ROW, d_pos=POS, d_ws=WS, ws_bytes=1 << 20, d_x=X, D=100,
                d_xs=XS)


@pytest.mark.parametrize("bad, why", [
    (dict(S=0), "S <="), (dict(S=(1 << 20) + 1), "S <="), (dict(K=0), "K <="), (dict(K=17), "K <="), (dict(E=0), "E <="),
    (dict(E=513), "E <="), (dict(d_eidx=0), "bad arguments"), (dict(d_offs=0), "bad arguments"),
    (dict(d_row=0), "bad arguments"), (dict(d_pos=0), "bad arguments"), (dict(d_ws=0), "bad arguments"),
    (dict(d_xs=0), "bad arguments"), (dict(d_eidx=IDS + 2), "misaligned"), (dict(d_offs=OFFS + 1), "misaligned"),
    (dict(d_row=ROW + 2), "misaligned"), (dict(d_pos=POS + 3), "misaligned"), (dict(d_ws=WS + 2), "misaligned"),
    (dict(S=5000, ws_bytes=100), "workspace"), (dict(ws_bytes=0), "workspace"), (dict(dtype=2), "dtype"),
    (dict(dtype=-1), "dtype"), (dict(D=0), "D <="), (dict(D=8193), "D <="), (dict(ldx=99), "closer"), (dict(ldxs=99), "closer"),
    (dict(ldx=-100), "closer"), (dict(ldxs=(1 << 36) + 1), "closer"), (dict(d_x=X + 2), "misaligned"),
    (dict(d_xs=XS + 2), "misaligned"), (dict(d_x=X + 1, dtype=1), "misaligned"),
    (dict(d_pos=IDS), "overlaps"), (dict(d_row=POS + 16), "overlaps"), (dict(d_offs=IDS + 64), "overlaps"),
    (dict(d_ws=POS + 4), "overlaps"), (dict(d_xs=X + 160), "overlaps"), (dict(d_xs=IDS), "overlaps"), (dict(d_row=XS), "overlaps"),
    (dict(d_offs=X), "overlaps"),
])
def test_dispatch_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.experts_dispatch_dev(**{**DISPATCH, **bad})


BACK = dict(d_y=XS, d_pos=POS, d_w=W, S=300, K=4, D=100, d_out=OUT, d_res=X)


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=2), "dtype"), (dict(S=0), "S <="), (dict(S=(1 << 20) + 1), "S <="), (dict(K=0), "K <="), (dict(K=17), "K <="),
    (dict(D=0), "D <="), (dict(D=8193), "D <="), (dict(d_y=0), "bad arguments"), (dict(d_pos=0), "bad arguments"),
    (dict(d_out=0), "bad arguments"), (dict(ldy=99), "closer"), (dict(ldr=99), "closer"), (dict(ldo=99), "closer"),
    (dict(ldo=-1), "closer"), (dict(d_y=XS + 2), "misaligned"), (dict(d_res=X + 2), "misaligned"),
    (dict(d_out=OUT + 1), "misaligned"), (dict(d_pos=POS + 2), "misaligned"), (dict(d_w=W + 1), "misaligned"),
    (dict(d_out=OUT + 1, dtype=1), "misaligned"), (dict(d_out=XS), "overlaps"), (dict(d_out=POS), "overlaps"),
    (dict(d_w=OUT + 400), "overlaps"), (dict(d_res=OUT + 4), "overlaps"), (dict(d_res=OUT, ldr=120), "overlaps"),
])
def test_back_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.experts_back_dev(**{**BACK, **bad})


GRAD = dict(d_dout=X, d_y=XS, d_pos=POS, d_w=W, S=300, K=4, D=100, d_dy=OUT, d_dw=Q)


@pytest.mark.parametrize("bad, why", [
    (dict(dtype=3), "dtype"), (dict(S=0), "S <="), (dict(K=17), "K <="), (dict(D=8193), "D <="), (dict(d_dout=0), "bad arguments"),
    (dict(d_y=0), "bad arguments"), (dict(d_pos=0), "bad arguments"), (dict(d_dy=0), "bad arguments"), (dict(ldg=99), "closer"),
    (dict(ldy=99), "closer"), (dict(lddy=99), "closer"), (dict(d_dout=X + 2), "misaligned"), (dict(d_y=XS + 2), "misaligned"),
    (dict(d_dy=OUT + 2), "misaligned"), (dict(d_dw=Q + 2), "misaligned"), (dict(d_w=W + 2), "misaligned"),
    (dict(d_pos=POS + 2), "misaligned"), (dict(d_dy=X), "overlaps"), (dict(d_dy=XS + 4), "overlaps"),
    (dict(d_dy=XS, lddy=120), "overlaps"), (dict(d_dw=W), "overlaps"), (dict(d_dw=OUT + 4), "overlaps"), (dict(d_dw=POS), "overlaps"),
    (dict(d_dy=W), "overlaps"), (dict(d_dw=XS), "overlaps"),
])
def test_back_grad_declines(bad, why):
    with pytest.raises(RuntimeError, match=why):
        zz.experts_back_grad_dev(**{**GRAD, **bad})


def test_tables_decline():
    for E, O, I in ((0, 8, 8), (513, 8, 8), (1, 0, 8), (1, 8, 0), (2, (1 << 24) + 1, 8), (2, 8, (1 << 16) + 1),
                    (1, 1 << 20, 1 << 15), (512, 1 << 16, 1 << 14)):
        for gated in (False, True):
            with pytest.raises(RuntimeError, match="bad shape"):
                zz.Fp8Experts(E, O, I, gated)
    L = zz.lib()
    c, s = np.zeros((8, 8), np.uint8), np.ones((1, 1), np.float32)
    assert L.zz_fp8_upload_expert(-1, 0, 0, None, None) == 0 and "bad arguments" in zz.last_error()
    assert L.zz_fp8_upload_expert(-1, 0, 0, c.ctypes.data_as(zz._u8p), s.ctypes.data_as(zz._f32p)) == 0
    assert L.zz_fp8_upload_expert_dev(-1, 0, 0, Q, SC + 2) == 0 and "bad arguments" in zz.last_error()
    assert L.zz_fp8_upload_expert_dev(-1, 0, 0, Q, SC) == 0


EP = dict(q=Q, s=SC, S=4, bias=W, act=1, clamp=0.0, res=X, ldr=0, dtype=0, y=Y, ldy=0)
BAD_EP = [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(act=3), "activation"), (dict(act=-1), "activation"),
    (dict(clamp=-1.0), "clamp"), (dict(clamp=NAN), "clamp"), (dict(clamp=INF), "clamp"), (dict(q=None), "bad arguments"),
    (dict(s=None), "bad arguments"), (dict(y=None), "bad arguments"), (dict(ldy=-1), "bad arguments"),
    (dict(ldr=-1), "bad arguments"), (dict(ldy=(1 << 36) + 1), "bad arguments"), (dict(q=Q + 8), "misaligned"),
    (dict(s=SC + 2), "misaligned"), (dict(y=Y + 2), "misaligned"), (dict(y=Y + 1, dtype=1), "misaligned"),
    (dict(res=X + 2), "misaligned"), (dict(bias=W + 2), "misaligned"),
]


@pytest.mark.parametrize("bad, why", BAD_EP + [(dict(S=0), "S <="), (dict(S=(1 << 20) + 1), "S <="), ({}, "gpu_init|no such")])
def test_epilogue_declines(bad, why):
    a = {**EP, **bad}
    assert zz.lib().zz_fp8_matmul_ep_dev(-1, a["q"], a["s"], a["S"], a["bias"], a["act"], a["clamp"], a["res"], a["ldr"],
                                         a["dtype"], a["y"], a["ldy"], None) == 0
    assert any(w in zz.last_error() for w in why.split("|")), zz.last_error()


@pytest.mark.parametrize("bad, why", BAD_EP + [
    (dict(S=0), "P, R"), (dict(S=(1 << 24) + 1, R=1 << 24, row=ROW), "P, R"), (dict(R=0), "P, R"), (dict(R=(1 << 24) + 1), "P, R"),
    (dict(offs=None), "P, R"), (dict(R=3), "R >= P"), (dict(row=ROW + 2), "misaligned"), (dict(offs=OFFS + 1), "misaligned"),
    ({}, "gpu_init|no such"),
])
def test_experts_product_declines(bad, why):
    a = {**EP, "R": 4, "row": None, "offs": OFFS, **bad}
    assert zz.lib().zz_fp8_matmul_experts_dev(-1, a["q"], a["s"], a["R"], a["row"], a["offs"], a["S"], a["bias"], a["act"],
                                              a["clamp"], a["res"], a["ldr"], a["dtype"], a["y"], a["ldy"], None) == 0
    assert any(w in zz.last_error() for w in why.split("|")), zz.last_error()
