"""8-bit rows and the fp8 product on the GPU against their 64-bit forms (zzref8.py)."""
import numpy as np
import pytest
import torch

import zzref8 as R
import zunzuncito_amd as zz

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
KIND = {F32: zz.ZZ_F32, BF16: zz.ZZ_BF16}


@pytest.fixture(autouse=True, scope="module")
def _up():
    zz.init()


def stream():
    return torch.cuda.current_stream().cuda_stream


def inputs(S, D, dtype, seed, wide=1):
    g = torch.Generator().manual_seed(seed)
    col = 1 + 30 * (torch.rand(D * wide, generator=g) < 0.02)
    x = (torch.randn(S, D * wide, generator=g) * col).to(dtype)
    res = (3 * torch.randn(S, D * wide, generator=g) * col).to(dtype)
    return x, res, 1 + 0.3 * torch.randn(D, generator=g)


def buffers(S, D):
    nb = R.blocks(D)
    # a row behind the last one, and a guard, that have to stay as they are
    return (torch.full((S + 1, nb * 128), 0x55, dtype=torch.uint8, device="cuda"),
            torch.full((nb * S + 3,), -7.0, device="cuda"))


def taken(q, s, S, D):
    torch.cuda.synchronize()
    assert bool((q[S] == 0x55).all()) and bool((s[-3:] == -7.0).all())
    return q[:S].cpu(), s[:-3].view(-1, S).cpu()


# one element, a block less one, a block, block edges, every number of groups a thread holds,
# odd widths (rows that no vector load fits), the largest
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, D", [(1, 1), (3, 7), (1, 127), (2, 128), (5, 129), (1, 2816), (4, 2048), (3, 2049),
                                  (2, 4095), (65, 1088), (1, 8192), (2, 8191), (130, 64)])
def test_add_norm(dtype, S, D):
    print("case", S, D, dtype, flush=True)
    x, res, w = inputs(S, D, dtype, 100 + S + D)
    X, Rs, Wt = x.cuda(), res.cuda(), w.cuda()
    for use_res, use_w, store in ((True, True, True), (False, True, False), (True, False, False)):
        q, s = buffers(S, D)
        sm = torch.full((S + 1, D), -5.0, dtype=dtype, device="cuda")
        zz.add_norm_fp8_dev(X.data_ptr(), Rs.data_ptr() if use_res else 0, sm.data_ptr() if store else 0,
                            Wt.data_ptr() if use_w else 0, S, D, 1e-6, q.data_ptr(), s.data_ptr(), KIND[dtype],
                            stream=stream())
        qh, sh = taken(q, s, S, D)
        h, y = R.norm_rows(x, res if use_res else None, w if use_w else None, float(np.float32(1e-6)))
        R.check_rows(y, qh, sh, R.norm_delta(D))
        if store:
            got = sm[:S].cpu()
            assert torch.equal(got, torch.from_numpy(h).float().to(dtype))     # h is f32's own: one rounding
        assert bool((sm[S if store else 0:] == -5.0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [5, 300, 2816])
def test_add_norm_range(dtype, D):
    """Rows whose squares 32 bits do not hold, with and without eps."""
    x, _, w = inputs(6, D, dtype, D)
    x = (x.float() * torch.tensor([1e-38, 1e-30, 1e-18, 1.0, 1e19, 1e36])[:, None]).to(dtype)
    X, Wt = x.cuda(), w.cuda()
    for eps in (0.0, 1e-6):
        q, s = buffers(6, D)
        zz.add_norm_fp8_dev(X.data_ptr(), 0, 0, Wt.data_ptr(), 6, D, eps, q.data_ptr(), s.data_ptr(), KIND[dtype],
                            stream=stream())
        qh, sh = taken(q, s, 6, D)
        h, y = R.norm_rows(x, None, w, float(np.float32(eps)))
        assert np.isfinite(y).all()
        R.check_rows(y, qh, sh, R.norm_delta(D))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D, ldx, off", [(2816, 5632, 0), (200, 203, 0), (256, 512, 1), (129, 160, 3)])
def test_add_norm_strides_and_in_place(dtype, D, ldx, off):
    """Rows apart, a start that no vector load fits, sum stored over res and over x."""
    S = 9
    g = torch.Generator().manual_seed(D)
    xb = torch.randn(S * ldx + off, generator=g).to(dtype)
    rb = torch.randn(S * ldx + off, generator=g).to(dtype)
    w = 1 + 0.1 * torch.randn(D, generator=g)
    for over in ("x", "res"):
        X, Rs, Wt = xb.cuda(), rb.cuda(), w.cuda()
        esz = X.element_size()
        px, pr = X.data_ptr() + off * esz, Rs.data_ptr() + off * esz
        q, s = buffers(S, D)
        zz.add_norm_fp8_dev(px, pr, px if over == "x" else pr, Wt.data_ptr(), S, D, 1e-5, q.data_ptr(), s.data_ptr(),
                            KIND[dtype], ldx=ldx, ldr=ldx, lds=ldx, stream=stream())
        qh, sh = taken(q, s, S, D)
        x = xb[off:].view(S, ldx)[:, :D]
        r = rb[off:].view(S, ldx)[:, :D]
        h, y = R.norm_rows(x, r, w, float(np.float32(1e-5)))
        R.check_rows(y, qh, sh, R.norm_delta(D))
        want = (xb if over == "x" else rb).clone()
        want[off:].view(S, ldx)[:, :D] = torch.from_numpy(h).float().to(dtype)
        assert torch.equal((X if over == "x" else Rs).cpu(), want)             # and nothing between the rows
        assert torch.equal((Rs if over == "x" else X).cpu(), rb if over == "x" else xb)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, D, ldx", [(1, 1, 1), (7, 130, 130), (33, 2112, 4224), (2, 20000, 20000), (1000, 64, 67),
                                       (5, 1088, 1088)])
def test_rows(dtype, S, D, ldx):
    g = torch.Generator().manual_seed(S * D)
    xb = (torch.randn(S * ldx, generator=g) * torch.exp(3 * torch.randn(S * ldx, generator=g))).to(dtype)
    X = xb.cuda()
    q, s = buffers(S, D)
    zz.rows_fp8_dev(X.data_ptr(), S, D, q.data_ptr(), s.data_ptr(), KIND[dtype], ldx=ldx, stream=stream())
    qh, sh = taken(q, s, S, D)
    R.check_rows(xb.view(S, ldx)[:, :D].double().numpy(), qh, sh, 0.0)


def test_rows_at_the_edges():
    """Zero blocks, values below the floor, the largest finite ones, subnormal codes; a NaN
    and an infinity stay in their rows."""
    x = torch.zeros(8, 256)
    x[1, :] = 2.0 ** -130
    x[2, :128] = torch.finfo(F32).max
    x[3, 0], x[3, 1:] = 448.0, torch.linspace(2.0 ** -11, 2.0 ** -5, 255)
    x[6] = 1.0
    clean = x.double().numpy()
    x[4, 5] = float("nan")
    x[5, 9] = float("inf")
    X = x.cuda()
    q, s = buffers(8, 256)
    zz.rows_fp8_dev(X.data_ptr(), 8, 256, q.data_ptr(), s.data_ptr(), stream=stream())
    qh, sh = taken(q, s, 8, 256)
    keep = [0, 1, 2, 3, 6, 7]
    R.check_rows(clean[keep], qh[keep], sh[:, keep], 0.0)
    v = R.e4m3_value(qh.numpy())
    assert np.isnan(v[4, 5]) and not np.isnan(np.delete(v[4], 5)).any()
    assert torch.isinf(sh[0, 5]) and np.isnan(v[5, 9]) and not np.isnan(v[5, 128:]).any()


def coded(shape, seed, lo=0, hi=256):
    """Codes of every finite kind."""
    r = np.random.default_rng(seed)
    c = r.integers(lo, hi, shape).astype(np.uint8)
    return np.where((c & 127) == 127, 3, c).astype(np.uint8)


def case(S, O, I, seed):
    r = np.random.default_rng(seed)
    xq = np.zeros((S, R.blocks(I) * 128), np.uint8)
    xq[:, :I] = coded((S, I), seed)
    xs = np.exp(r.normal(-5, 1, (R.blocks(I), S))).astype(np.float32)
    wq = coded((O, I), seed + 1)
    ws = np.exp(r.normal(-8, 1, (R.blocks(O), R.blocks(I)))).astype(np.float32)
    return xq, xs, wq, ws


# one of everything, ragged tiles in each direction, block edges of the matrix's scales, and
# sizes at which each of the kernel's forms is the one chosen
SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 129), (1, 2816, 2112), (3, 1000, 1088), (16, 129, 300), (17, 128, 2816),
          (21, 1000, 1088), (33, 257, 511), (64, 704, 2816), (65, 2112, 640), (100, 130, 1000), (128, 256, 256),
          (200, 1500, 700), (256, 512, 128), (300, 257, 1025), (513, 640, 2816), (700, 2816, 704), (1025, 300, 130),
          (300, 2000, 1100), (2100, 2050, 200), (2500, 2500, 300), (385, 4697, 603), (1441, 4314, 131),
          (1025, 4161, 1025), (3651, 3351, 386), (900, 9043, 1323)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, O, I", SHAPES)
def test_product(dtype, S, O, I):
    print("case", S, O, I, dtype, flush=True)
    xq, xs, wq, ws = case(S, O, I, S + O + I)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(wq, ws)
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        y = torch.full((S + 1, O), -3.0, dtype=dtype, device="cuda")
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), KIND[dtype], stream=stream())
        torch.cuda.synchronize()
        assert bool((y[S] == -3.0).all())
        want, mag = R.product(xq, xs, wq, ws, O, I)
        got = y[:S].double().cpu().numpy()
        off = np.abs(got - want)
        assert np.all(off <= R.product_bound(mag, want, I, dtype)), (off / np.maximum(mag, 1e-300)).max()
        again = torch.empty_like(y[:S])
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, again.data_ptr(), KIND[dtype], stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(again, y[:S])
    finally:
        m.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, O, I, ldy, off", [(5, 130, 200, 133, 0), (40, 130, 200, 200, 1), (300, 130, 200, 136, 0),
                                               (300, 130, 200, 131, 3), (300, 2000, 1100, 2008, 0), (700, 2816, 704, 2817, 5),
                                               (1500, 1500, 600, 1504, 8), (2100, 2050, 200, 2051, 1),
                                               (2500, 2500, 300, 2501, 0), (385, 4697, 603, 4703, 3),
                                               (1025, 4161, 700, 4164, 4), (3651, 3351, 386, 3353, 1)])
def test_product_strides(dtype, S, O, I, ldy, off):
    print("case", S, O, I, ldy, off, dtype, flush=True)
    xq, xs, wq, ws = case(S, O, I, 5)
    m = zz.Fp8Matrix(O, I)
    try:
        D = [torch.from_numpy(a).cuda() for a in (xq, xs, wq, ws)]
        torch.cuda.synchronize()
        m.upload_dev(D[2].data_ptr(), D[3].data_ptr())
        y = torch.full((S * ldy + off,), -3.0, dtype=dtype, device="cuda")
        m.matmul_dev(D[0].data_ptr(), D[1].data_ptr(), S, y.data_ptr() + off * y.element_size(), KIND[dtype], ldy=ldy,
                     stream=stream())
        v = y[off:].view(S, ldy).double().cpu().numpy()
        want, mag = R.product(xq, xs, wq, ws, O, I)
        assert np.all(np.abs(v[:, :O] - want) <= R.product_bound(mag, want, I, dtype))
        assert np.all(v[:, O:] == -3.0) and bool((y[:off] == -3.0).all())
    finally:
        m.close()


@pytest.mark.parametrize("S, O, I", [(70, 300, 300), (300, 2000, 1100), (700, 2816, 704), (1500, 1500, 600),
                                     (2100, 2050, 200), (2500, 2500, 300), (385, 4697, 603), (1025, 4161, 700),
                                     (3651, 3351, 386)])
def test_product_rows_apart(S, O, I):
    """A row of NaN codes and one of infinite scales touch no other row, in every form."""
    print("case", S, O, I, flush=True)
    xq, xs, wq, ws = case(S, O, I, 8)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(wq, ws)
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        ys = [torch.empty(S, O, device="cuda") for _ in range(2)]
        for y, bad in zip(ys, (False, True)):
            if bad:
                Q[S // 2, I - 1] = 0xFF
                Sc[0, S - 1] = float("inf")
            m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        keep = torch.ones(S, dtype=torch.bool)
        keep[[S // 2, S - 1]] = False
        assert torch.equal(ys[0][keep.cuda()], ys[1][keep.cuda()])
        assert bool(ys[1][S // 2].isnan().all()) and not bool(ys[1][S - 1].isfinite().any())
    finally:
        m.close()


def test_product_edges():
    """Row independence (a NaN row, an infinite scale), the largest codes, a second upload, a
    matrix without weights, and the host form."""
    S, O, I = 37, 140, 260
    xq, xs, wq, ws = case(S, O, I, 77)
    m = zz.Fp8Matrix(O, I)
    try:
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        y = torch.full((S, O), -3.0, device="cuda")
        with pytest.raises(RuntimeError, match="no weights"):
            m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        with pytest.raises(RuntimeError, match="no weights"):
            m.matmul(np.ones((2, I), np.float32))
        m.upload(wq, ws)
        with pytest.raises(RuntimeError, match="closer"):
            m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), ldy=O - 1, stream=stream())
        with pytest.raises(RuntimeError, match="overlaps"):
            m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, Q.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert bool((y == -3.0).all())
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        Q2, Sc2 = Q.clone(), Sc.clone()
        Q2[3, 7] = 0x7F
        Sc2[1, 20] = float("inf")
        y2 = torch.empty_like(y)
        m.matmul_dev(Q2.data_ptr(), Sc2.data_ptr(), S, y2.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        other = [t for t in range(S) if t not in (3, 20)]
        assert torch.equal(y2[other], y[other]) and bool(y2[3].isnan().all()) and not bool(y2[20].isfinite().any())
        # 448 * 448 * I, exact in f32's 24 bits for one block
        full = np.full((O, I), 0x7E, np.uint8)
        m.upload(full, np.ones_like(ws))
        Q.fill_(0)
        Q[:, :I] = 0x7E
        Sc.fill_(1.0)
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert bool((y == 448.0 * 448.0 * I).all())
        # the host form is the two device calls
        m.upload(wq, ws)
        x = np.random.default_rng(1).normal(size=(S, I)).astype(np.float32)
        X = torch.from_numpy(x).cuda()
        zz.rows_fp8_dev(X.data_ptr(), S, I, Q.data_ptr(), Sc.data_ptr(), stream=stream())
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert np.array_equal(m.matmul(x), y.cpu().numpy())
    finally:
        m.close()


def test_two_matrices_streams_and_graphs():
    """Matrices beside each other on two streams, and a captured chain (norm, product, rows,
    product) replayed with eager work between: every replay is the eager result."""
    S, D, M = 19, 320, 200
    a, b = zz.Fp8Matrix(M, D), zz.Fp8Matrix(D, M)
    try:
        _, _, wa, sa = case(1, M, D, 3)
        _, _, wb, sb = case(1, D, M, 4)
        a.upload(wa, sa)
        b.upload(wb, sb)
        g = torch.Generator(device="cuda").manual_seed(6)
        w = torch.ones(D, device="cuda")

        class Run:
            def __init__(self):
                self.x = torch.empty(S, D, device="cuda")
                self.res = torch.empty(S, D, device="cuda")
                self.q, self.s = torch.empty(S, 384, dtype=torch.uint8, device="cuda"), torch.empty(3, S, device="cuda")
                self.h = torch.empty(S, M, dtype=BF16, device="cuda")
                self.q2, self.s2 = torch.empty(S, 256, dtype=torch.uint8, device="cuda"), torch.empty(2, S, device="cuda")
                self.sum, self.y = torch.empty(S, D, device="cuda"), torch.empty(S, D, device="cuda")

            def __call__(self):
                st = stream()
                zz.add_norm_fp8_dev(self.x.data_ptr(), self.res.data_ptr(), self.sum.data_ptr(), w.data_ptr(), S, D,
                                    1e-6, self.q.data_ptr(), self.s.data_ptr(), stream=st)
                a.matmul_dev(self.q.data_ptr(), self.s.data_ptr(), S, self.h.data_ptr(), zz.ZZ_BF16, stream=st)
                zz.rows_fp8_dev(self.h.data_ptr(), S, M, self.q2.data_ptr(), self.s2.data_ptr(), zz.ZZ_BF16, stream=st)
                b.matmul_dev(self.q2.data_ptr(), self.s2.data_ptr(), S, self.y.data_ptr(), stream=st)

        one, two, eager = Run(), Run(), Run()
        graphs = []
        torch.cuda.synchronize()
        for r in (one, two):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                r()
            graphs.append(gr)
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        for k in range(4):
            for r in (one, two):
                r.x.normal_(generator=g)
                r.res.normal_(generator=g)
            torch.cuda.synchronize()
            for st, gr in zip(side, graphs):
                with torch.cuda.stream(st):
                    gr.replay()
            torch.cuda.synchronize()
            for r in (one, two):
                eager.x.copy_(r.x)
                eager.res.copy_(r.res)
                eager()
                torch.cuda.synchronize()
                assert torch.equal(eager.y, r.y) and torch.equal(eager.sum, r.sum), k
    finally:
        a.close()
        b.close()


@pytest.mark.parametrize("S", [3, 20])
def test_product_large_matrix(S):
    """A matrix past the caches (64 MiB and more), against its own rows in a small one and
    against 64 bits for some of them."""
    O, I = 65600, 1088
    g = torch.Generator(device="cuda").manual_seed(S)
    wq = torch.randint(0, 127, (O, I), generator=g, dtype=torch.uint8, device="cuda")
    wq += (torch.rand(O, I, generator=g, device="cuda") < 0.5).to(torch.uint8) * 128
    ws = torch.rand(R.blocks(O), R.blocks(I), generator=g, device="cuda")
    xq, xs, _, _ = case(S, 1, I, S)
    Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
    m = zz.Fp8Matrix(O, I)
    try:
        torch.cuda.synchronize()
        m.upload_dev(wq.data_ptr(), ws.data_ptr())
        y = torch.full((S + 1, O), -3.0, device="cuda")
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert bool((y[S] == -3.0).all())
        for at, n in ((0, 128), (33 * 128, 256), (O - 64, 64)):
            part = wq[at:at + n].cpu().numpy()
            sc = ws[at // 128:at // 128 + R.blocks(n)].cpu().numpy()
            want, mag = R.product(xq, xs, part, sc, n, I)
            off = np.abs(y[:S, at:at + n].double().cpu().numpy() - want)
            assert np.all(off <= R.product_bound(mag, want, I, F32))
    finally:
        m.close()


def test_rows_and_product_past_32_bits():
    """The most rows, at offsets that 32 bits do not hold: norm, rounding and product of the
    first, the last and some between against 64 bits."""
    S, D, O = 1 << 20, 2200, 40
    at = [0, 1, S // 2 - 1, S - 33, S - 1]
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(S, D, dtype=BF16, device="cuda").normal_(generator=g)
    sm = torch.empty_like(x)
    nb = R.blocks(D)
    q = torch.empty(S, nb * 128, dtype=torch.uint8, device="cuda")
    s = torch.empty(nb, S, device="cuda")
    zz.add_norm_fp8_dev(x.data_ptr(), x.data_ptr(), sm.data_ptr(), 0, S, D, 1e-6, q.data_ptr(), s.data_ptr(), zz.ZZ_BF16,
                        stream=stream())
    torch.cuda.synchronize()
    xh = x[at].cpu()
    h, y = R.norm_rows(xh, xh, None, float(np.float32(1e-6)))
    R.check_rows(y, q[at].cpu(), s[:, at].cpu(), R.norm_delta(D))
    assert torch.equal(sm[at].cpu(), torch.from_numpy(h).float().to(BF16))
    zz.rows_fp8_dev(x.data_ptr(), S, D, q.data_ptr(), s.data_ptr(), zz.ZZ_BF16, stream=stream())
    torch.cuda.synchronize()
    R.check_rows(xh.double().numpy(), q[at].cpu(), s[:, at].cpu(), 0.0)
    _, _, wq, ws = case(1, O, D, 6)
    m = zz.Fp8Matrix(O, D)
    try:
        m.upload(wq, ws)
        out = torch.empty(S, O, device="cuda")
        m.matmul_dev(q.data_ptr(), s.data_ptr(), S, out.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        want, mag = R.product(q[at].cpu().numpy(), s[:, at].cpu().numpy(), wq, ws, O, D)
        assert np.all(np.abs(out[at].double().cpu().numpy() - want) <= R.product_bound(mag, want, D, F32))
    finally:
        m.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 7, 9, 500, 511, 513, 1023, 1025, 2047, 4097])
def test_rows_of_other_widths(dtype, D):
    """Few threads a row and many, rows that share a workgroup, a last group that reads on into
    the next row: what follows a row's end, and the buffer's, is NaN."""
    for S in (1, 2, 3, 5):
        x, res, w = inputs(S, D, dtype, 7 * S + D, 2)
        nan = torch.full((1,), float("nan"), dtype=dtype)
        x[:, D:], res[:, D:] = nan, nan
        X, Rs, Wt = (torch.cat([t.view(-1).to(t.dtype), torch.full((64,), float("nan"), dtype=t.dtype)]).cuda() for t in (x, res, w))
        q, s = buffers(S, D)
        sm = torch.full((S, 2 * D), -5.0, dtype=dtype, device="cuda")
        zz.add_norm_fp8_dev(X.data_ptr(), Rs.data_ptr(), sm.data_ptr(), Wt.data_ptr(), S, D, 1e-6, q.data_ptr(), s.data_ptr(),
                            KIND[dtype], ldx=2 * D, ldr=2 * D, lds=2 * D, stream=stream())
        qh, sh = taken(q, s, S, D)
        h, y = R.norm_rows(x[:, :D], res[:, :D], w, float(np.float32(1e-6)))
        R.check_rows(y, qh, sh, R.norm_delta(D))
        assert torch.equal(sm[:, :D].cpu(), torch.from_numpy(h).float().to(dtype)) and bool((sm[:, D:] == -5.0).all())
        q, s = buffers(S, D)
        zz.rows_fp8_dev(X.data_ptr(), S, D, q.data_ptr(), s.data_ptr(), KIND[dtype], ldx=2 * D, stream=stream())
        qh, sh = taken(q, s, S, D)
        R.check_rows(x[:, :D].double().numpy(), qh, sh, 0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, O, I, ldy", [(4200, 4100, 140, 4160), (8300, 4104, 200, 4104)])
def test_product_large_result(dtype, S, O, I, ldy):
    """Results of 64 MiB and more, whose lines tiles write whole and those they do not."""
    xq, xs, wq, ws = case(S, O, I, 9)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(wq, ws)
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        y = torch.full((S, ldy), -3.0, dtype=dtype, device="cuda")
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), KIND[dtype], ldy=ldy, stream=stream())
        torch.cuda.synchronize()
        assert bool((y[:, O:] == -3.0).all())
        want, mag = R.product(xq, xs, wq, ws, O, I)
        off = np.abs(y[:, :O].double().cpu().numpy() - want)
        assert np.all(off <= R.product_bound(mag, want, I, dtype))
    finally:
        m.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["normal", "small integers", "halves of steps", "magnitudes"])
def test_rows_exact(dtype, kind):
    """Scales and codes to the last bit, at ties too: values of few bits lie right between two
    codes often, and a quotient that is off by a bit takes the odd one."""
    S, D = 301, 2100
    g = torch.Generator().manual_seed(len(kind))
    x = torch.randn(S, D, generator=g)
    if kind == "small integers":
        x = torch.randint(-57, 58, (S, D), generator=g).float()
    elif kind == "halves of steps":                      # 448 the largest: all other values between two codes
        x = torch.randint(16, 31, (S, D), generator=g).float() + 0.5
        x = x * torch.exp2(torch.randint(-12, 4, (S, D), generator=g).float()) * (1 - 2 * torch.randint(0, 2, (S, D), generator=g))
        x[:, ::128] = 448.0
        x[:, -1] = -448.0
        x = x * torch.exp2(torch.randint(-30, 31, (S, 1), generator=g).float())
    elif kind == "magnitudes":                           # from below the floor to the largest, block by block
        e = torch.linspace(-126, 124, S)[:, None].round()
        x = x.clamp(-7.9, 7.9) * torch.exp2(e)
    x = x.to(dtype)
    x[7, 130:140] = -0.0
    X = x.cuda()
    q, s = buffers(S, D)
    zz.rows_fp8_dev(X.data_ptr(), S, D, q.data_ptr(), s.data_ptr(), KIND[dtype], stream=stream())
    qh, sh = taken(q, s, S, D)
    want, scale = R.rows_exact(x.float().numpy())
    assert np.array_equal(sh.numpy(), scale)
    got = R.e4m3_value(qh.numpy())
    assert np.array_equal(got, want), (np.count_nonzero(got != want), got.size)
    assert np.array_equal(qh.numpy()[:, :D] >> 7, np.signbit(x.float().numpy()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [3, 128, 1000, 2816, 8192])
def test_add_norm_ends_of_range(dtype, D):
    """Rows at both ends of the type, subnormal ones too, whose reciprocal root 32 bits do not
    hold; without eps they are as good as any."""
    S = 6
    g = torch.Generator().manual_seed(D)
    x = (0.5 + 0.5 * torch.rand(S, D, generator=g)) * (1 - 2 * torch.randint(0, 2, (S, D), generator=g))
    x = (x.double() * torch.tensor([2.0 ** -129, 2.0 ** -132, 2.0 ** -140, 1.0, 2.0 ** 127, 1.99 * 2.0 ** 127])[:, None].double()).float()
    x[2, 0] = 2.0 ** -133                                # bf16 holds no smaller one
    x = x.to(dtype)
    w = 1 + 0.3 * torch.randn(D, generator=g)
    X, Wt = x.cuda(), w.cuda()
    for wt, use in ((w, Wt.data_ptr()), (None, 0)):
        q, s = buffers(S, D)
        zz.add_norm_fp8_dev(X.data_ptr(), 0, 0, use, S, D, 0.0, q.data_ptr(), s.data_ptr(), KIND[dtype], stream=stream())
        qh, sh = taken(q, s, S, D)
        _, y = R.norm_rows(x, None, wt, 0.0)
        assert np.isfinite(y).all() and np.abs(y).max() > 0.1
        R.check_rows(y, qh, sh, R.norm_delta(D))


def product_on(xq, xs, wq, ws, O, I, dtype):
    """R.product and R.product_bound of a large result, in 64 bits on the device."""
    x = torch.from_numpy(R.e4m3_value(xq)[:, :I] * np.repeat(xs.astype(np.float64).T, 128, 1)[:, :I]).cuda()
    w = R.e4m3_value(wq) * np.repeat(np.repeat(ws.astype(np.float64), 128, 0)[:O], 128, 1)[:, :I]
    w = torch.from_numpy(np.ascontiguousarray(w.T)).cuda()
    want, mag = x @ w, x.abs() @ w.abs()
    return want, R.product_bound(mag, 0.0, I, dtype) + R.HALF[dtype] * want.abs()


# results of 64 MiB and more whose lines tiles write whole, which are stored past the caches: for
# each type 64 x 128 and 128 x 128 tiles, and both with what is over a round in parts; no size a
# tile divides
@pytest.mark.parametrize("dtype, S, O, I, ldy", [
    (F32, 8331, 2002, 129, 2016), (F32, 8903, 2066, 129, 2080), (F32, 2584, 7445, 515, 7456), (F32, 2949, 6845, 777, 6848),
    (BF16, 4870, 6927, 129, 6944), (BF16, 7299, 4577, 129, 4608), (BF16, 6190, 6472, 513, 6496),
    (BF16, 7041, 5281, 643, 5312)])
def test_product_past_the_caches(dtype, S, O, I, ldy):
    print("case", S, O, I, ldy, dtype, flush=True)
    xq, xs, wq, ws = case(S, O, I, S)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(wq, ws)
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        y = torch.full((S + 1, ldy), -3.0, dtype=dtype, device="cuda")
        assert y.data_ptr() % 64 == 0 and ldy * y.element_size() % 64 == 0 and S * ldy * y.element_size() >= 64 << 20
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), KIND[dtype], ldy=ldy, stream=stream())
        torch.cuda.synchronize()
        assert bool((y[:, O:] == -3.0).all()) and bool((y[S] == -3.0).all())
        want, lim = product_on(xq, xs, wq, ws, O, I, dtype)
        assert bool(((y[:S, :O].double() - want).abs_() <= lim).all())
    finally:
        m.close()


@pytest.mark.parametrize("S, O, I, dtype", [(1, 65600, 1088, BF16), (8, 65600, 1088, BF16), (9, 65600, 1088, BF16),
                                            (32, 65600, 1088, BF16), (5, 65600, 1200, F32), (32, 18432, 7168, BF16)])
def test_product_large_matrices(S, O, I, dtype):
    """Matrices past the caches, all of the result: in 16 bits, in both forms that are stored
    past them, at both ends of their rows; with more columns, where another form is chosen."""
    r = np.random.default_rng(S)
    xq, xs, _, _ = case(S, 1, I, S)
    wq = coded((O, I), S)
    ws = np.exp(r.normal(-8, 1, (R.blocks(O), R.blocks(I)))).astype(np.float32)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(wq, ws)
        Q, Sc = torch.from_numpy(xq).cuda(), torch.from_numpy(xs).cuda()
        y = torch.full((S + 1, O), -3.0, dtype=dtype, device="cuda")
        m.matmul_dev(Q.data_ptr(), Sc.data_ptr(), S, y.data_ptr(), KIND[dtype], stream=stream())
        torch.cuda.synchronize()
        assert bool((y[S] == -3.0).all())
        want, lim = product_on(xq, xs, wq, ws, O, I, dtype)
        assert bool(((y[:S].double() - want).abs_() <= lim).all())
    finally:
        m.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [500, 1000, 2000, 2816, 5035])
def test_add_norm_past_the_caches(dtype, D):
    """A sum of 64 MiB and a few rows, with each number of threads and groups a row: all of the
    sum, and some rows' codes."""
    S = (64 << 20) // (D * (4 if dtype == F32 else 2)) + 3
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(S, D, generator=g, device="cuda").to(dtype)
    res = torch.randn(S, D, generator=g, device="cuda").to(dtype)
    w = 1 + 0.3 * torch.randn(D, generator=g, device="cuda")
    q, s = buffers(S, D)
    sm = torch.full((S + 1, D), -5.0, dtype=dtype, device="cuda")
    zz.add_norm_fp8_dev(x.data_ptr(), res.data_ptr(), sm.data_ptr(), w.data_ptr(), S, D, 1e-6, q.data_ptr(), s.data_ptr(),
                        KIND[dtype], stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(sm[:S], (x.float() + res.float()).to(dtype)) and bool((sm[S] == -5.0).all())
    qh, sh = taken(q, s, S, D)
    at = [*range(9), S // 3, S // 2, *range(S - 9, S)]
    _, y = R.norm_rows(x[at].cpu(), res[at].cpu(), w.cpu(), float(np.float32(1e-6)))
    R.check_rows(y, qh[at], sh[:, at], R.norm_delta(D))
