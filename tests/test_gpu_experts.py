"""Tokens to experts and back, the gradient, the product's epilogue and the experts' products on
the GPU against their 64-bit forms (zzrefx.py, zzref8.py)."""
import numpy as np
import pytest
import torch

import zzref8 as R
import zzrefx as X
import zunzuncito_amd as zz

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
KIND = {F32: zz.ZZ_F32, BF16: zz.ZZ_BF16}
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True, scope="module")
def _up():
    zz.init()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return 0 if t is None else t.data_ptr()


def routing(S, K, E, kind, seed):
    """ids [S, K]: distinct in a token (as a router's), any, all one expert's, with dropped ones."""
    g = torch.Generator().manual_seed(seed)
    if kind == "top" and K <= E:
        ids = torch.rand(S, E, generator=g).topk(K, dim=1)[1]
    elif kind == "one":
        ids = torch.full((S, K), E - 1)
    elif kind == "none":
        ids = torch.full((S, K), -1)
    else:
        ids = torch.randint(0, E, (S, K), generator=g)
    ids = ids.int()
    if kind == "dropped":
        wild = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31, E + 64], dtype=torch.int32)
        at = torch.rand(S, K, generator=g) < 0.3
        ids[at] = wild[torch.randint(0, 5, (int(at.sum()),), generator=g)]
    return ids


def rows(n, D, dtype, seed, ld=None, size=1.0):
    """A strided device view [n, D] of normal values and its buffer."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((n, ld or D), 77.0, dtype=dtype)
    buf[:, :D] = (size * torch.randn(n, D, generator=g)).to(dtype)
    return buf.cuda()


def dispatch(ids, E, x=None, D=0, dtype=F32, ldx=0, ldxs=0, ws=None):
    """The call with guards behind every output; what it must leave is left at -9 (rows: 55)."""
    S, K = ids.shape
    n = S * K
    I = ids.cuda()
    offs = torch.full((E + 3,), -9, dtype=torch.int32, device="cuda")
    row, pos = (torch.full((n + 2,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    need = zz.experts_ws_bytes(S, K, E)
    ws = torch.full((need + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    xs = torch.full((n + 1, ldxs or max(D, 1)), 55.0, dtype=dtype, device="cuda")
    zz.experts_dispatch_dev(ptr(I), S, K, E, ptr(offs), ptr(row), ptr(pos), ptr(ws), need, d_x=ptr(x), D=D,
                            d_xs=ptr(xs) if x is not None else 0, dtype=KIND[dtype], ldx=ldx, ldxs=ldxs, stream=stream())
    torch.cuda.synchronize()
    assert (offs[E + 1:] == -9).all() and (row[n:] == -9).all() and (pos[n:] == -9).all()
    assert (ws[need:] == 0x5A).all()
    return offs[:E + 1].cpu(), row[:n].cpu(), pos[:n].view(S, K).cpu(), xs.cpu()


def check_dispatch(ids, E, got):
    offs, row, pos, xs = got
    o, r, p = X.sort(ids.numpy(), E)
    assert np.array_equal(offs.numpy(), o) and np.array_equal(pos.numpy(), p)
    assert np.array_equal(row.numpy()[:r.size], r) and (row.numpy()[r.size:] == -9).all()
    return r


# one pair, a decode token, the edges of the one-launch form (1024 pairs) and of the sort by one
# workgroup (8192), several chunks, one expert and all of them, more choices than experts
@pytest.mark.parametrize("kind", ["top", "any", "one", "none", "dropped"])
@pytest.mark.parametrize("S, K, E, D", [(1, 1, 1, 1), (1, 8, 128, 2816), (3, 16, 512, 9), (37, 4, 32, 129), (128, 8, 512, 65),
                                        (1024, 1, 3, 4), (1025, 1, 64, 33), (129, 8, 65, 17), (1024, 8, 256, 7),
                                        (1025, 8, 128, 40), (3000, 16, 511, 3), (20011, 3, 2, 2)])
def test_dispatch(S, K, E, D, kind):
    for dtype in (F32, BF16):
        print("case", S, K, E, D, kind, dtype, flush=True)
        ids = routing(S, K, E, kind, S + K)
        x = rows(S, D, dtype, 5)
        got = dispatch(ids, E, x, D, dtype)
        r = check_dispatch(ids, E, got)
        xs = got[3]
        assert torch.equal(xs[:r.size].view(torch.uint8), x.cpu()[torch.from_numpy(r)].view(torch.uint8))
        assert (xs[r.size:] == 55.0).all()


def test_dispatch_without_rows():
    for S, K, E in ((5, 2, 9), (700, 4, 100), (5000, 4, 77)):
        ids = routing(S, K, E, "dropped", 3)
        check_dispatch(ids, E, dispatch(ids, E))


# every remainder of 16 bytes, rows that begin at any element, gaps between them
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, K", [(7, 3), (600, 3)])
def test_dispatch_strides(S, K, dtype):
    for D, ldx, ldxs, off in ((1, 3, 5, 1), (5, 5, 7, 2), (9, 11, 9, 3), (15, 16, 17, 1), (131, 133, 140, 7), (8192, 8193, 8192, 1)):
        print("case", S, K, D, dtype, flush=True)
        ids = routing(S, K, 11, "any", D)
        buf = rows(1, off + S * ldx, dtype, D).view(-1)
        x = buf[off:].view(S, ldx)
        n = S * K
        out = torch.full((off + (n + 1) * ldxs,), 55.0, dtype=dtype, device="cuda")
        xs = out[off:].view(n + 1, ldxs)
        I = ids.cuda()
        offs, row, pos = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (12, n, n))
        ws = torch.empty(zz.experts_ws_bytes(S, K, 11), dtype=torch.uint8, device="cuda")
        zz.experts_dispatch_dev(ptr(I), S, K, 11, ptr(offs), ptr(row), ptr(pos), ptr(ws), ws.numel(), d_x=x.data_ptr(), D=D,
                                d_xs=xs.data_ptr(), dtype=KIND[dtype], ldx=ldx, ldxs=ldxs, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(xs[:n, :D], x[row.long(), :D])
        assert (xs[:n, D:] == 55.0).all() and (xs[n] == 55.0).all() and (out[:off] == 55.0).all()


def test_dispatch_bits():
    """Rows are copied, not converted: NaNs keep their bits, minus zero its sign."""
    for dtype, it in ((F32, torch.int32), (BF16, torch.int16)):
        x = torch.randint(-2 ** 15, 2 ** 15, (40, 64), generator=torch.Generator().manual_seed(1)).to(it)
        x[0, :3] = torch.tensor([0x7f81, -0x7f, -0x8000]).to(it)
        for S in (3, 40):
            ids = routing(S, 16, 30, "any", 2)
            _, row, _, xs = dispatch(ids, 30, x[:S].cuda().view(dtype), 64, dtype)
            assert torch.equal(xs[:S * 16].view(it), x[row.long()])


def test_dispatch_largest():
    """16 million pairs; then rows whose elements pass 2^31."""
    S, K, E = 1 << 20, 16, 512
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(-1, E, (S, K), generator=g, dtype=torch.int32, device="cuda")
    offs, row, pos = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (E + 1, S * K, S * K))
    ws = torch.empty(zz.experts_ws_bytes(S, K, E), dtype=torch.uint8, device="cuda")
    zz.experts_dispatch_dev(ptr(ids), S, K, E, ptr(offs), ptr(row), ptr(pos), ptr(ws), ws.numel(), stream=stream())
    flat = ids.view(-1).long()
    kept = torch.nonzero(flat >= 0)[:, 0]
    order = kept[torch.sort(flat[kept], stable=True)[1]]
    assert torch.equal(row[:order.numel()].long(), order // K)
    want = torch.full_like(flat, -1)
    want[order] = torch.arange(order.numel(), device="cuda")
    assert torch.equal(pos.long(), want) and int(offs[E]) == order.numel()
    del want, order, kept, flat, ids
    S, K, D, ldxs = 40000, 8, 64, 8192
    ids = torch.randint(0, E, (S, K), generator=g, dtype=torch.int32, device="cuda")
    x = torch.randn(S, D, generator=g, device="cuda").to(BF16)
    xs = torch.zeros(S * K, ldxs, dtype=BF16, device="cuda")
    row, pos = row[:S * K], pos[:S * K]
    zz.experts_dispatch_dev(ptr(ids), S, K, E, ptr(offs), ptr(row), ptr(pos), ptr(ws), ws.numel(), d_x=ptr(x), D=D, d_xs=ptr(xs),
                            dtype=KIND[BF16], ldxs=ldxs, stream=stream())
    assert torch.equal(xs[:, :D], x[row.long()])
    out = torch.empty(S, D, dtype=BF16, device="cuda")
    w = torch.full((S, K), 0.125, device="cuda")                     # eight eighths of a row are the row
    zz.experts_back_dev(ptr(xs), ptr(pos), ptr(w), S, K, D, ptr(out), dtype=KIND[BF16], ldy=ldxs, stream=stream())
    assert torch.equal(out, x)
    dw = torch.empty(S, K, device="cuda")
    zz.experts_back_grad_dev(ptr(x), ptr(xs), ptr(pos), 0, S, K, D, ptr(xs), ptr(dw), dtype=KIND[BF16], ldy=ldxs, lddy=ldxs,
                             stream=stream())
    assert torch.equal(xs[:, :D], x[row.long()])                     # in place: what was there already
    sq = x.double().square().sum(1, keepdim=True)
    assert (dw - sq).abs().max() <= (X.dw_bound(1.0, D) * sq).max()


# ------------------------------------------------------------------ the way back and its gradient
SHAPES = [(1, 1, 1), (1, 8, 2816), (3, 16, 1087), (21, 8, 129), (50, 3, 8192), (300, 2, 64), (64, 16, 7), (5, 9, 4095), (700, 8, 40)]


def permuted(S, K, seed, drop):
    """pos [S, K]: distinct positions, a part of the pairs without one (a whole token's among them)."""
    g = torch.Generator().manual_seed(seed)
    pos = torch.randperm(S * K, generator=g).int().view(S, K)
    if drop:
        at = torch.rand(S, K, generator=g) < 0.25
        at[S // 2] = True
        wild = torch.tensor([-1, S * K, 2 ** 31 - 1, -2 ** 31, -5], dtype=torch.int32)
        pos[at] = wild[torch.randint(0, 5, (int(at.sum()),), generator=g)]
    return pos


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, K, D", SHAPES)
def test_back(S, K, D, dtype):
    print("case", S, K, D, dtype, flush=True)
    for drop, weighted, res, gap in ((False, True, True, 0), (True, True, False, 3), (True, False, True, 1), (False, False, False, 0)):
        pos = permuted(S, K, D, drop)
        y, r = rows(S * K, D, dtype, 7, D + gap), rows(S, D, dtype, 8, D + 2 * gap, 2.0)
        w = torch.rand(S, K, generator=torch.Generator().manual_seed(9)) - 0.3
        ok = (pos >= 0) & (pos < S * K)
        if drop:                                 # what is not read may be anything
            free = torch.ones(S * K, dtype=torch.bool)
            free[pos[ok].long()] = False
            y[free.cuda()] = NAN
            w[~ok] = NAN
        out = torch.full((S + 1, D + gap), 33.0, dtype=dtype, device="cuda")
        want, mag = X.back(y[:, :D].float().cpu().numpy(), pos.numpy(), w.numpy() if weighted else None,
                           r[:, :D].float().cpu().numpy() if res else None)
        P, W = pos.cuda(), w.cuda()
        zz.experts_back_dev(ptr(y), ptr(P), ptr(W) if weighted else 0, S, K, D, ptr(out), d_res=ptr(r) if res else 0,
                            dtype=KIND[dtype], ldy=D + gap, ldr=D + 2 * gap, ldo=D + gap, stream=stream())
        got = out.float().cpu().numpy()
        bound = X.back_bound(want, mag, K, R.HALF[dtype])
        assert np.all(np.abs(got[:S, :D] - want) <= bound)
        assert (got[S] == 33.0).all() and (got[:, D:] == 33.0).all()
        if res:                                  # onto the residual itself
            zz.experts_back_dev(ptr(y), ptr(P), ptr(W) if weighted else 0, S, K, D, ptr(r), d_res=ptr(r), dtype=KIND[dtype],
                                ldy=D + gap, ldr=D + 2 * gap, ldo=D + 2 * gap, stream=stream())
            assert torch.equal(r[:, :D], out[:S, :D]) and (r[:, D:] == 77.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S, K, D", SHAPES)
def test_back_grad(S, K, D, dtype):
    print("case", S, K, D, dtype, flush=True)
    for drop, weighted, gap in ((False, True, 0), (True, True, 3), (True, False, 1)):
        pos = permuted(S, K, D, drop)
        y, g = rows(S * K, D, dtype, 17, D + gap), rows(S, D, dtype, 18, D + 2 * gap)
        w = torch.rand(S, K, generator=torch.Generator().manual_seed(9)) - 0.3
        ok = (pos >= 0) & (pos < S * K)
        free = torch.ones(S * K, dtype=torch.bool)
        free[pos[ok].long()] = False
        y[free.cuda()] = NAN
        w[~ok] = NAN
        dy = torch.full((S * K + 1, D + gap), 33.0, dtype=dtype, device="cuda")
        dw = torch.full((S * K + 1,), 33.0, device="cuda")
        P, W = pos.cuda(), w.cuda()
        args = dict(dtype=KIND[dtype], ldg=D + 2 * gap, ldy=D + gap, lddy=D + gap, stream=stream())
        zz.experts_back_grad_dev(ptr(g), ptr(y), ptr(P), ptr(W) if weighted else 0, S, K, D, ptr(dy), ptr(dw), **args)
        want, wdw, mag = X.grad(g[:, :D].float().cpu().numpy(), y[:, :D].float().cpu().numpy(), pos.numpy(),
                                w.numpy() if weighted else None)
        got, half = dy.float().cpu().numpy(), R.HALF[dtype]
        for p, v in want.items():
            assert np.all(np.abs(got[p, :D] - v) <= (X.U + half * (1 + X.U)) * np.abs(v))
        assert (got[:-1][free.numpy()] == 33.0).all() and (got[-1] == 33.0).all() and (got[:, D:] == 33.0).all()
        gw = dw.cpu().numpy()
        assert np.all(np.abs(gw[:-1].reshape(S, K) - wdw) <= X.dw_bound(mag, D)) and gw[-1] == 33.0
        alone = torch.full_like(dy, 33.0)        # dy without dw, y unread
        zz.experts_back_grad_dev(ptr(g), 0, ptr(P), ptr(W) if weighted else 0, S, K, D, ptr(alone), 0, **args)
        assert torch.equal(alone, dy)
        zz.experts_back_grad_dev(ptr(g), ptr(y), ptr(P), ptr(W) if weighted else 0, S, K, D, ptr(y), ptr(dw), **args)
        kept = torch.nonzero(~free)[:, 0].cuda()                     # dy over y
        assert torch.equal(y[kept, :D], dy[kept, :D]) and np.array_equal(dw.cpu().numpy(), gw)


def test_gradients_against_differences():
    """<dout, back(y, w)> is linear in w and in y, <dxs, dispatch(x)> in x: a difference over any
    step is the gradient, up to the roundings of the two results (bounds as test_back's)."""
    S, K, E, D = 12, 3, 5, 70
    ids = routing(S, K, E, "dropped", 6)
    x, g = rows(S, D, F32, 1), rows(S, D, F32, 2)
    n = S * K
    offs, row, pos = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (E + 1, n, n))
    ws = torch.empty(64, dtype=torch.uint8, device="cuda")
    I = ids.cuda()
    xs = torch.zeros(n, D, device="cuda")

    def spread(v):
        xs.zero_()
        zz.experts_dispatch_dev(ptr(I), S, K, E, ptr(offs), ptr(row), ptr(pos), ptr(ws), 64, d_x=ptr(v), D=D, d_xs=ptr(xs), stream=stream())
        return xs.double().cpu()

    def back(y, w):
        out = torch.empty(S, D, device="cuda")
        zz.experts_back_dev(ptr(y), ptr(pos), ptr(w), S, K, D, ptr(out), stream=stream())
        return float((out.double() * g.double()).sum())

    spread(x)
    y, w = rows(n, D, F32, 3), torch.rand(S, K, generator=torch.Generator().manual_seed(5)).cuda()
    dy, dw = torch.zeros_like(y), torch.empty(S, K, device="cuda")
    zz.experts_back_grad_dev(ptr(g), ptr(y), ptr(pos), ptr(w), S, K, D, ptr(dy), ptr(dw), stream=stream())
    kept = int(offs[E])
    G, Y = g.double().abs().cpu().numpy(), y.double().abs().cpu().numpy()
    rng = np.random.default_rng(7)
    for _ in range(12):
        s, j = int(rng.integers(S)), int(rng.integers(K))
        up, dn = w.clone(), w.clone()
        up[s, j] += 0.5
        dn[s, j] -= 0.5
        p = int(pos.view(S, K)[s, j])
        _, mag = X.back(Y, pos.view(S, K).cpu().numpy(), (w.abs() + 0.5).cpu().numpy(), None)
        off = 2 * (X.back_bound(mag, mag, K, R.HALF[F32]) * G).sum() + X.dw_bound((G[s] * Y[max(p, 0)]).sum(), D)
        step = float(up[s, j]) - float(dn[s, j])
        assert abs((back(y, up) - back(y, dn)) / step - float(dw[s, j])) <= off / step + 1e-12
        p, d = int(rng.integers(kept)), int(rng.integers(D))
        up, dn = y.clone(), y.clone()
        up[p, d] += 1.0
        dn[p, d] -= 1.0
        step = float(up[p, d]) - float(dn[p, d])
        _, mag = X.back(Y + 1.0, pos.view(S, K).cpu().numpy(), w.cpu().numpy(), None)
        off = 2 * (X.back_bound(mag, mag, K, R.HALF[F32]) * G).sum()
        assert abs((back(up, w) - back(dn, w)) / step - float(dy[p, d])) <= off / step + X.U * abs(float(dy[p, d]))
    dxs = rows(n, D, F32, 4)
    dx = torch.empty(S, D, device="cuda")
    zz.experts_back_dev(ptr(dxs), ptr(pos), 0, S, K, D, ptr(dx), stream=stream())
    H = dxs.double().cpu()
    for _ in range(12):
        s, d = int(rng.integers(S)), int(rng.integers(D))
        up, dn = x.clone(), x.clone()
        up[s, d] += 1.0
        dn[s, d] -= 1.0
        step = float(up[s, d]) - float(dn[s, d])
        diff = ((spread(up) - spread(dn)) * H)[:kept].sum() / step      # the copies are exact
        at = pos.view(S, K)[s]
        mag = H[at[at >= 0].long().cpu(), d].abs().sum()
        assert abs(float(diff) - float(dx[s, d])) <= (K + 1) * X.U * float(mag) + 1e-12


@pytest.mark.parametrize("dtype, S, D", [(F32, 3000, 8192), (BF16, 9001, 4099)])
def test_way_past_the_caches(dtype, S, D):
    """Rows of 64 MiB and more, which are stored past the caches: copies, a sum of two rows and the
    gradient, whose values are exact or of one rounding."""
    K = 2
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(S, D, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, 40, (S, K), generator=g, device="cuda", dtype=torch.int32)
    n = S * K
    offs, row, pos = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (41, n, n))
    ws = torch.empty(zz.experts_ws_bytes(S, K, 40), dtype=torch.uint8, device="cuda")
    xs = torch.full((n + 1, D), 7.0, dtype=dtype, device="cuda")
    zz.experts_dispatch_dev(ptr(ids), S, K, 40, ptr(offs), ptr(row), ptr(pos), ptr(ws), ws.numel(), d_x=ptr(x), D=D, d_xs=ptr(xs),
                            dtype=KIND[dtype], stream=stream())
    assert torch.equal(xs[:n], x[row.long()]) and (xs[n] == 7.0).all()
    out = torch.full((S + 1, D), 7.0, dtype=dtype, device="cuda")
    zz.experts_back_dev(ptr(xs), ptr(pos), 0, S, K, D, ptr(out), d_res=ptr(x), dtype=KIND[dtype], stream=stream())
    assert torch.equal(out[:S], (x.float() + x.float() + x.float()).to(dtype)) and (out[S] == 7.0).all()
    w = torch.rand(S, K, generator=g, device="cuda")
    dy = torch.full((n + 1, D), 7.0, dtype=dtype, device="cuda")
    zz.experts_back_grad_dev(ptr(x), 0, ptr(pos), ptr(w), S, K, D, ptr(dy), 0, dtype=KIND[dtype], stream=stream())
    p = pos.view(S, K).long()
    for j in range(K):
        assert torch.equal(dy[p[:, j]], (w[:, j:j + 1] * x.float()).to(dtype))
    assert (dy[n] == 7.0).all()


# ------------------------------------------------------------------ products
def codes(shape, seed, small=False):
    """e4m3 codes without NaN; small: of magnitude up to 2, so that sums reach the activations' bend."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 64 if small else 127, shape, generator=g, dtype=torch.uint8)
    return c + (torch.rand(shape, generator=g) < 0.5).to(torch.uint8) * 128


def scales(shape, seed, size):
    g = torch.Generator().manual_seed(seed)
    return size * (0.5 + torch.rand(shape, generator=g))


class Case:
    """A table of experts (E = 1 for one matrix), rows, bias and residual, on both sides."""

    def __init__(self, E, O, I, gated, rows_, P, seed, dtype=F32, bias=True, res=True, size=1.0):
        G, nb, no = 2 if gated else 1, R.blocks(I), R.blocks(O)
        self.E, self.O, self.I, self.G, self.dtype = E, O, I, G, dtype
        self.wq, self.ws = codes((E, G, O, I), seed, True), scales((E, G, no, nb), seed + 1, size / np.sqrt(I))
        self.xq = codes((rows_, nb * 128), seed + 2, True)
        self.xq[:, I:] = 0
        self.xs = scales((nb, rows_), seed + 3, 1.0)
        self.bias = torch.randn(E, G, O, generator=torch.Generator().manual_seed(seed + 4)) if bias else None
        self.res = rows(P, O, dtype, seed + 5) if res else None
        self.mat = zz.Fp8Experts(E, O, I, gated)
        for e in range(E):
            for p in range(G):
                if (e + p) % 2:
                    a, b = self.wq[e, p].cuda(), self.ws[e, p].cuda()
                    torch.cuda.synchronize()
                    self.mat.upload_dev(e, ptr(a), ptr(b), part=p)
                else:
                    self.mat.upload(e, self.wq[e, p].numpy(), self.ws[e, p].numpy(), part=p)
        self.q, self.s, self.b = self.xq.cuda(), self.xs.cuda(), self.bias.cuda() if bias else None

    def want(self, e, at, out, act, clamp, bias=True, res=True, cols=None):
        """(y, bound) of expert e's product of the rows `at`, which are rows `out` of y; cols: of whole
        blocks of 128 columns alone, a slice"""
        cols = cols or slice(0, self.O)
        n, blocks = cols.stop - cols.start, slice(cols.start // 128, R.blocks(cols.stop))
        xq, xs = self.xq[at].numpy(), self.xs[:, at].numpy()
        w = [(xq, xs, self.wq[e, p, cols].numpy(), self.ws[e, p, blocks].numpy(), n, self.I) for p in range(self.G)]
        sums, mags = zip(*(R.product(*a) for a in w))
        b = self.bias[e][:, cols].numpy() if bias and self.bias is not None else None
        r = self.res[out.cuda()][:, cols].float().cpu().numpy() if res and self.res is not None else None
        # results in bf16 may come from the 8-bit instructions
        cut = [X.eights(*a) for a in w] if self.dtype == BF16 else [0.0, 0.0]
        return X.epilogue(sums, mags, self.I, b, act, clamp, r, R.HALF[self.dtype], cut)


def near(got, want, bound):
    got = got.double().cpu().numpy()
    off = np.abs(got - want)
    assert np.all(off <= bound), (np.nanmax(off / bound), np.argwhere(~(off <= bound))[:4])
    # all in all the rounding to bf16 (half a step is 2^-8 at most) is what shows
    assert np.linalg.norm(off) <= (2.0 ** -8 + 2.0 ** -10) * np.linalg.norm(want)


ACTS = [(zz.ZZ_EP_NONE, 0.0), (zz.ZZ_EP_GELU_TANH, 0.0), (zz.ZZ_EP_SILU, 0.0)]


# a single row and column, ragged edges of blocks and groups, each form's sizes
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("S, O, I", [(1, 1, 1), (1, 16, 128), (2, 17, 129), (3, 15, 300), (1, 2816, 2112), (8, 1000, 704),
                                     (33, 31, 257), (65, 33, 1088), (100, 1000, 512), (130, 129, 640), (300, 704, 300),
                                     (520, 515, 256), (1000, 2112, 128), (2100, 1056, 257),
                                     (1300, 1409, 384), (129, 4224, 130)])
def test_epilogue(S, O, I, gated):
    for dtype in (F32, BF16):
        print("case", S, O, I, gated, dtype, flush=True)
        c = Case(1, O, I, gated, S, S, S + O + I, dtype, size=0.3)
        try:
            for act, clamp, b, r in ((0, 0.0, True, True), (1, 0.0, True, False), (2, 0.7 if gated else 0.0, False, True)):
                y = torch.full((S + 1, O), 9.0, dtype=dtype, device="cuda")
                c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), d_bias=ptr(c.b) if b else 0, act=act, clamp=clamp,
                                    d_res=ptr(c.res) if r else 0, dtype=KIND[dtype], stream=stream())
                at = torch.arange(S) if S <= 130 else torch.cat([torch.arange(40), torch.arange(S - 40, S), torch.arange(60, S, 17)])
                near(y[at.cuda()], *c.want(0, at, at, act, clamp, b, r))
                assert (y[S] == 9.0).all()
                again = torch.empty_like(y)
                c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(again), d_bias=ptr(c.b) if b else 0, act=act, clamp=clamp,
                                    d_res=ptr(c.res) if r else 0, dtype=KIND[dtype], stream=stream())
                assert torch.equal(y[:S], again[:S])
        finally:
            c.mat.close()


def picked(n, k=12):
    """The first rows, the last and some between."""
    return torch.arange(n) if n <= 3 * k else torch.unique(torch.cat([torch.arange(k), torch.arange(n - k, n), torch.arange(k, n, n // k)]))


# sizes that between them take every form that a product's rows, columns and type choose from, with
# three blocks of columns at least, and matrices that are read past the caches
@pytest.mark.parametrize("dtype, gated, S, O, I", [
    (F32, False, 34, 4169, 576), (F32, False, 480, 4146, 385), (F32, False, 65, 5447, 796), (F32, False, 517, 1973, 257),
    (F32, False, 361, 1352, 514), (F32, False, 1090, 3600, 257), (F32, False, 736, 4157, 259), (F32, True, 1, 4247, 529),
    (F32, True, 137, 5631, 392), (F32, True, 37, 4162, 810), (F32, True, 33, 4284, 649), (F32, True, 37, 4234, 526),
    (F32, True, 518, 3466, 260), (F32, True, 455, 3107, 263), (BF16, False, 1764, 1194, 263), (BF16, False, 1926, 1555, 259),
    (BF16, False, 1239, 5017, 260), (BF16, False, 33, 4212, 533), (BF16, False, 326, 5533, 291), (BF16, False, 66, 5540, 813),
    (BF16, False, 66, 5769, 561), (BF16, True, 265, 3817, 258), (BF16, True, 262, 5067, 257), (BF16, True, 641, 4548, 259),
    (BF16, True, 145, 5608, 279), (BF16, True, 35, 4114, 808), (BF16, True, 35, 4220, 529), (F32, False, 3, 65600, 1088),
    (F32, False, 20, 65600, 1088), (BF16, True, 3, 32800, 1088), (BF16, True, 20, 32800, 1088)])
def test_epilogue_in_every_form(dtype, gated, S, O, I):
    print("case", S, O, I, gated, dtype, flush=True)
    c = Case(1, O, I, gated, S, S, S + O + I, dtype, size=0.3)
    try:
        act, clamp = (2, 0.8) if gated else (1, 0.0)
        y = torch.full((S + 1, O), 9.0, dtype=dtype, device="cuda")
        c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), d_bias=ptr(c.b), act=act, clamp=clamp, d_res=ptr(c.res),
                            dtype=KIND[dtype], stream=stream())
        at = picked(S)
        for lo in (0, O // 256 * 128, O // 128 * 128):
            cols = slice(lo, min(lo + 256, O))
            near(y[at.cuda()][:, cols], *c.want(0, at, at, act, clamp, cols=cols))
        assert (y[S] == 9.0).all()
    finally:
        c.mat.close()


# each tile's rounds, which go in threes and keep the scales of 64 blocks, at their ends
@pytest.mark.parametrize("nb", [1, 2, 3, 4, 5, 65, 67])
@pytest.mark.parametrize("gated, S, O", [(False, 2401, 1031), (False, 610, 4897), (False, 2182, 2691), (True, 641, 1930),
                                         (True, 898, 1682), (True, 2182, 1346)])
def test_epilogue_in_tiles_of_any_depth(gated, S, O, nb):
    I = 128 * nb - 3
    c = Case(1, O, I, gated, S, S, S + nb, BF16, size=0.3, res=False)
    try:
        y = torch.full((S + 1, O), 9.0, dtype=BF16, device="cuda")
        c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), d_bias=ptr(c.b), act=2, dtype=KIND[BF16], stream=stream())
        at = picked(S)
        for lo in (0, O // 128 * 128):
            cols = slice(lo, min(lo + 128, O))
            near(y[at.cuda()][:, cols], *c.want(0, at, at, 2, 0.0, cols=cols))
        assert (y[S] == 9.0).all()
    finally:
        c.mat.close()


# as above, for tables of experts and a skewed spread of the rows
@pytest.mark.parametrize("dtype, gated, E, P, O, I", [
    (F32, False, 53, 55, 1802, 713), (F32, False, 137, 195, 34, 609), (F32, False, 51, 3492, 143, 667), (F32, False, 38, 1235, 213, 770),
    (F32, False, 26, 851, 291, 586), (F32, False, 428, 1965, 139, 280), (F32, False, 6, 395, 4274, 263), (F32, True, 17, 17, 2646, 752),
    (F32, True, 44, 3190, 72, 606), (F32, True, 8, 36, 4324, 267), (F32, True, 38, 2504, 321, 317), (BF16, False, 222, 242, 462, 657),
    (BF16, False, 302, 1300, 213, 259), (BF16, False, 344, 3885, 180, 314), (BF16, False, 31, 2019, 1774, 267),
    (BF16, False, 68, 2274, 100, 555), (BF16, True, 11, 11, 3736, 828), (BF16, True, 13, 55, 2628, 266),
    (BF16, True, 259, 3277, 116, 376), (BF16, True, 45, 3158, 518, 292), (BF16, True, 5, 323, 1655, 258)])
def test_experts_in_every_form(dtype, gated, E, P, O, I):
    print("case", E, P, O, I, gated, dtype, flush=True)
    n = max(1, P // 2)
    c = Case(E, O, I, gated, n, P, E + P, dtype, size=0.4)
    try:
        offs = spread(P, E, "skew", E + P)
        at = torch.randint(0, n, (P,), generator=torch.Generator().manual_seed(P))
        row, D = at.int().cuda(), offs.cuda()
        act, clamp = (1, 0.0) if gated else (2, 0.0)
        y = torch.full((P + 1, O), 9.0, dtype=dtype, device="cuda")
        c.mat.matmul_dev(ptr(c.q), ptr(c.s), n, ptr(row), ptr(D), P, ptr(y), d_bias=ptr(c.b), act=act, d_res=ptr(c.res),
                         dtype=KIND[dtype], stream=stream())
        o = offs.tolist()
        some = [e for e in range(E) if o[e] < o[e + 1]]
        for e in some[:3] + some[-3:] + some[3:-3:max(1, len(some) // 12)]:
            out = o[e] + picked(o[e + 1] - o[e])
            lo = max(0, (O - 1) // 128 * 128 - 128) if e % 2 else 0
            cols = slice(lo, min(lo + 256, O))
            near(y[out.cuda()][:, cols], *c.want(e, at[out], out, act, clamp, cols=cols))
        assert (y[o[E]:] == 9.0).all()
    finally:
        c.mat.close()


@pytest.mark.parametrize("dtype, gated, S, O, I", [(F32, False, 4100, 4224, 130), (F32, True, 4100, 4224, 130),
                                                   (BF16, False, 8300, 4224, 130), (BF16, True, 8300, 4224, 130)])
def test_epilogue_large_result(dtype, gated, S, O, I):
    """Results of 64 MiB and more are stored past the caches where rows begin at whole lines, and
    are what they are elsewhere."""
    print("case", S, O, I, gated, dtype, flush=True)
    c = Case(1, O, I, gated, S, 1, 5, dtype, res=False)
    try:
        a = torch.full((S + 1, O), 9.0, dtype=dtype, device="cuda")
        b = torch.full(((S + 1) * O + 1,), 9.0, dtype=dtype, device="cuda")[1:].view(S + 1, O)
        for y in (a, b):
            c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, y.data_ptr(), d_bias=ptr(c.b), act=1, dtype=KIND[dtype], stream=stream())
        assert torch.equal(a, b) and (a[S] == 9.0).all()
        at = picked(S)
        near(a[at.cuda()][:, :256], *c.want(0, at, at, 1, 0.0, cols=slice(0, 256)))
    finally:
        c.mat.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("S, O, I", [(1, 100, 200), (40, 67, 300), (200, 131, 129), (700, 260, 128)])
def test_epilogue_strides_and_in_place(S, O, I, gated):
    """Rows apart, beginning at any element; the residual elsewhere and in y itself."""
    for dtype in (F32, BF16):
        for ldy, ldr, off in ((O, O, 1), (O + 3, O + 5, 3)):
            print("case", S, O, I, gated, dtype, ldy, flush=True)
            c = Case(1, O, I, gated, S, S, 7 + S, dtype)
            try:
                res = torch.full((off + S * ldr,), 5.0, dtype=dtype, device="cuda")
                v = res[off:].view(S, ldr)
                v[:, :O] = c.res
                out = torch.full((off + (S + 1) * ldy,), 9.0, dtype=dtype, device="cuda")
                y = out[off:].view(S + 1, ldy)
                args = dict(d_bias=ptr(c.b), act=1, clamp=0.5 if gated else 0.0, dtype=KIND[dtype], stream=stream())
                c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, y.data_ptr(), d_res=v.data_ptr(), ldr=ldr, ldy=ldy, **args)
                near(y[:S, :O], *c.want(0, torch.arange(S), torch.arange(S), 1, args["clamp"]))
                assert (y[:, O:] == 9.0).all() and (y[S] == 9.0).all() and (out[:off] == 9.0).all()
                c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, v.data_ptr(), d_res=v.data_ptr(), ldr=ldr, ldy=ldr, **args)
                assert torch.equal(v[:, :O], y[:S, :O]) and (v[:, O:] == 5.0).all()
            finally:
                c.mat.close()


def test_epilogue_of_a_plain_matrix():
    """zz_fp8_create's matrix takes the epilogue too; without one the sums are the plain product's."""
    S, O, I = 70, 200, 300
    c = Case(1, O, I, False, S, S, 3)
    m = zz.Fp8Matrix(O, I)
    try:
        m.upload(c.wq[0, 0].numpy(), c.ws[0, 0].numpy())
        y, z, p = (torch.empty(S, O, device="cuda") for _ in range(3))
        m.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), d_bias=ptr(c.b), act=2, d_res=ptr(c.res), stream=stream())
        c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(z), d_bias=ptr(c.b), act=2, d_res=ptr(c.res), stream=stream())
        assert torch.equal(y, z)
        m.matmul_dev(ptr(c.q), ptr(c.s), S, ptr(p), stream=stream())
        m.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), stream=stream())
        assert torch.equal(y, p)
    finally:
        c.mat.close()
        m.close()


@pytest.mark.parametrize("gated", [False, True])
def test_epilogue_edges(gated):
    """NaN codes, infinite scales, bias and residual: their own rows and columns only; sums far out
    on both sides of the activations; a clamp that everything passes."""
    for S in (2, 40, 200):
        O, I = 70, 128
        c = Case(1, O, I, gated, S, S, 11, bias=True, res=True)
        try:
            args = dict(d_bias=ptr(c.b), d_res=ptr(c.res), stream=stream())
            for act in (0, 1, 2):
                for clamp in ((0.0, 0.25) if gated else (0.0,)):
                    y, z = (torch.empty(S, O, device="cuda") for _ in range(2))
                    c.mat.matmul_ep_dev(ptr(c.q), ptr(c.s), S, ptr(y), act=act, clamp=clamp, **args)
                    q, s, b, r = c.q.clone(), c.s.clone(), c.b.clone(), c.res.clone()
                    q[1, 5], b[0, 0, 7], r[0, 9] = 0x7F, NAN, INF
                    if gated:
                        b[0, 1, 8] = NAN
                    c.mat.matmul_ep_dev(ptr(q), ptr(s), S, ptr(z), act=act, clamp=clamp, d_bias=ptr(b), d_res=ptr(r), stream=stream())
                    bad = torch.zeros(S, O, dtype=torch.bool, device="cuda")
                    bad[1], bad[:, 7] = True, True
                    if gated:
                        bad[:, 8] = True
                    assert z[bad].isnan().all() and z[0, 9] == INF
                    bad[0, 9] = True
                    assert torch.equal(z[~bad], y[~bad])
            # scales that put sums between 1e-30 and 1e30
            big = Case(1, O, I, gated, S, S, 12, bias=False, res=False)
            try:
                big.xs *= torch.logspace(-30, 30, S).view(1, S)
                big.s = big.xs.cuda()
                for act in (0, 1, 2):
                    y = torch.empty(S, O, device="cuda")
                    big.mat.matmul_ep_dev(ptr(big.q), ptr(big.s), S, ptr(y), act=act, clamp=3.0 if gated else 0.0, stream=stream())
                    assert y.isfinite().all()
                    near(y, *big.want(0, torch.arange(S), torch.arange(S), act, 3.0 if gated else 0.0))
            finally:
                big.mat.close()
        finally:
            c.mat.close()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("S, O, I", [(1764, 1194, 263), (1926, 1555, 259), (1239, 5017, 260), (517, 1973, 257)])
def test_epilogue_edges_in_tiles(S, O, I, gated):
    """The same in the tiles of larger products: a NaN code, bias or residual and an infinite scale
    stay in their row or column."""
    for dtype in (F32, BF16):
        print("case", S, O, I, gated, dtype, flush=True)
        c = Case(1, O, I, gated, S, S, 11, dtype)
        try:
            out = []
            q, s, b, r = c.q.clone(), c.s.clone(), c.b.clone(), c.res.clone()
            for k in range(2):
                y = torch.empty(S, O, dtype=dtype, device="cuda")
                c.mat.matmul_ep_dev(ptr(q), ptr(s), S, ptr(y), d_bias=ptr(b), act=2, clamp=0.5 if gated else 0.0, d_res=ptr(r),
                                    dtype=KIND[dtype], stream=stream())
                out.append(y)
                q[70, 5], b[0, 0, 133], r[9, 40], s[0, S - 1] = 0xFF, NAN, NAN, INF
            y, z = out
            bad = torch.zeros(S, O, dtype=torch.bool, device="cuda")
            bad[70], bad[:, 133], bad[9, 40] = True, True, True
            assert z[bad].isnan().all()
            bad[S - 1] = True
            assert torch.equal(z[~bad], y[~bad]) and y.isfinite().all()
        finally:
            c.mat.close()


def spread(P, E, kind, seed):
    """offs [E + 1] over at most P rows."""
    rng = np.random.default_rng(seed)
    if kind == "even":
        n = np.full(E, P // E)
    elif kind == "one":
        n = np.zeros(E, int)
        n[E // 2] = P
    elif kind == "empty":
        n = np.zeros(E, int)
    else:
        part = rng.random(E) ** 4 * (rng.random(E) < 0.7)
        n = np.floor(part / max(part.sum(), 1e-9) * P * 0.9).astype(int)
    o = np.concatenate([[0], np.cumsum(n)])
    if kind == "late":
        o += P - o[-1]
    return torch.from_numpy(o).int()


# decode's pairs, batches, prompts; one expert and 512; experts without rows, with all of them
@pytest.mark.parametrize("kind", ["even", "one", "skew", "late", "empty"])
@pytest.mark.parametrize("E, P, O, I, gated", [(1, 1, 1, 1, False), (8, 8, 704, 300, True), (128, 8, 33, 129, True),
                                               (5, 21, 70, 257, False), (512, 600, 16, 128, False), (65, 700, 40, 130, True),
                                               (9, 500, 130, 300, True), (4, 900, 515, 129, False), (16, 3000, 100, 256, True),
                                               (3, 2000, 520, 384, True), (3, 2500, 1100, 128, False)])
def test_experts(E, P, O, I, gated, kind):
    for dtype in (F32, BF16):
        for indexed in (False, True):
            print("case", E, P, O, I, gated, kind, dtype, indexed, flush=True)
            n = max(1, P // 3) if indexed else P + 2
            c = Case(E, O, I, gated, n, P, E + P, dtype, size=0.4)
            try:
                offs = spread(P, E, kind, E + P + 1)
                row = None
                at = torch.arange(P)
                if indexed:
                    at = torch.randint(0, n, (P,), generator=torch.Generator().manual_seed(P))
                    row = at.int()
                    wild = torch.rand(P, generator=torch.Generator().manual_seed(P + 1)) < 0.1
                    row[wild] = torch.tensor([-1, n, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.arange(int(wild.sum())) % 4]
                    at = torch.where(wild, 0, at)
                    row = row.cuda()
                D = offs.cuda()
                act, clamp = (2, 0.6) if gated else (1, 0.0)
                y = torch.full((P + 1, O), 9.0, dtype=dtype, device="cuda")
                c.mat.matmul_dev(ptr(c.q), ptr(c.s), n, ptr(row), ptr(D), P, ptr(y), d_bias=ptr(c.b), act=act, clamp=clamp,
                                 d_res=ptr(c.res), dtype=KIND[dtype], stream=stream())
                torch.cuda.synchronize()
                o = offs.tolist()
                for e in range(E):
                    if o[e] < o[e + 1]:
                        out = torch.arange(o[e], o[e + 1])
                        out = torch.unique(torch.cat([out[:33], out[-33:], out[::29]]))
                        near(y[out.cuda()], *c.want(e, at[out], out, act, clamp))
                assert (y[:o[0]] == 9.0).all() and (y[o[E]:] == 9.0).all()
            finally:
                c.mat.close()


@pytest.mark.parametrize("dtype, gated, E, P, O, I", [
    (F32, False, 39, 1265, 434, 261), (F32, True, 145, 172, 17, 534), (F32, True, 26, 865, 153, 790), (F32, True, 104, 3766, 65, 300),
    (F32, True, 91, 3045, 43, 538), (BF16, False, 145, 150, 39, 531), (BF16, False, 46, 3152, 131, 515), (BF16, False, 53, 1699, 149, 848),
    (BF16, True, 152, 152, 17, 534), (BF16, True, 91, 3296, 35, 872), (BF16, True, 74, 2726, 49, 529), (BF16, True, 13, 400, 700, 259)])
def test_experts_in_the_smaller_forms(dtype, gated, E, P, O, I):
    test_experts_in_every_form(dtype, gated, E, P, O, I)


@pytest.mark.parametrize("dtype, gated, E, P, O, I, ldy", [
    (F32, False, 3, 20, 70, 300, 1 << 28), (BF16, True, 3, 20, 70, 300, 1 << 28), (F32, True, 2, 700, 130, 260, 1 << 23),
    (BF16, False, 2, 700, 130, 260, 1 << 23), (F32, False, 2, 9000, 140, 130, 1 << 19), (BF16, True, 2, 9000, 140, 130, 1 << 19)])
def test_experts_far_rows(dtype, gated, E, P, O, I, ldy):
    """Rows of y whose elements pass 2^32, from few rows and in tiles."""
    assert P * ldy > 1 << 32
    c = Case(E, O, I, gated, P, P, 3, dtype, res=False)
    y = torch.empty(P, ldy, dtype=dtype, device="cuda")
    try:
        offs = [0] + [P // 3] * (E - 1) + [P]
        D = torch.tensor(offs, dtype=torch.int32).cuda()
        y[-1].fill_(9.0)
        for first in (True, False):              # then with itself as the residual
            if not first:
                y[:, :O] = torch.randn(P, O, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
                c.res = y[:, :O].clone()
            c.mat.matmul_dev(ptr(c.q), ptr(c.s), P, 0, ptr(D), P, ptr(y), d_bias=ptr(c.b), act=2, dtype=KIND[dtype], ldy=ldy,
                             d_res=0 if first else ptr(y), ldr=ldy, stream=stream())
            torch.cuda.synchronize()
            for e in (0, E - 1):
                at = torch.unique(torch.cat([torch.arange(offs[e], offs[e + 1])[k] for k in (slice(0, 3), slice(-4, None))]))
                near(y[at.cuda(), :O], *c.want(e, at, at, 2, 0.0))
            assert (y[-1, O:] == 9.0).all()
    finally:
        c.mat.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_experts_far_codes(dtype):
    """Codes of the rows, and of the table, that pass 2^32 bytes; the last of them."""
    I, O, E, P = 1 << 16, 33, 3, 70000
    c = Case(E, O, I, False, 256, 256, 6, dtype, res=False)
    q, s = c.q.repeat(P // 256 + 1, 1)[:P], c.s.repeat(1, P // 256 + 1)[:, :P].contiguous()
    y = torch.empty(P, O, dtype=dtype, device="cuda")
    try:
        assert q.numel() > 1 << 32
        offs = [0, 0, 100, P]
        D = torch.tensor(offs, dtype=torch.int32).cuda()
        c.mat.matmul_dev(ptr(q), ptr(s), P, 0, ptr(D), P, ptr(y), d_bias=ptr(c.b), act=1, dtype=KIND[dtype], stream=stream())
        torch.cuda.synchronize()
        for e, at in ((1, [0, 99]), (2, [100, 65535, 65536, P - 1])):
            at = torch.tensor(at)
            near(y[at.cuda()], *c.want(e, at % 256, at, 1, 0.0))
    finally:
        c.mat.close()
    del q, s, y
    O, E, P = 4096, 20, 45
    c = Case(1, O, I, False, P, P, 6, dtype, res=False)
    t = zz.Fp8Experts(E, O, I)
    try:
        zero, w, ws = torch.zeros(O, I, dtype=torch.uint8, device="cuda"), c.wq[0, 0].cuda(), c.ws[0, 0].cuda()
        torch.cuda.synchronize()
        for e in range(E):
            t.upload_dev(e, ptr(w if e == E - 1 else zero), ptr(ws))
        b = c.b.expand(E, 1, O).contiguous()
        y = torch.empty(P, O, dtype=dtype, device="cuda")
        for n in (2, P):                         # of the last expert; the others' are the bias alone
            D = torch.tensor([0] * 5 + [P - n] * 15 + [P], dtype=torch.int32).cuda()
            t.matmul_dev(ptr(c.q), ptr(c.s), P, 0, ptr(D), P, ptr(y), d_bias=ptr(b), dtype=KIND[dtype], stream=stream())
            torch.cuda.synchronize()
            at = torch.tensor([P - n, P - 1])
            cols = slice(O - 128, O)
            near(y[at.cuda(), cols], *c.want(0, at, at, 0, 0.0, cols=cols))
            assert torch.equal(y[:P - n], c.b.view(O).to(dtype).expand(P - n, O))
    finally:
        c.mat.close()
        t.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gated", [False, True])
def test_experts_most_rows(dtype, gated):
    """2^24 rows of 512 experts, and 2^20 of one matrix: codes of 1 and scales of whole numbers, exact."""
    E, P, O, I = 512, 1 << 24, 3, 5
    t = zz.Fp8Experts(E, O, I, gated)
    one = zz.Fp8Experts(1, O, I, gated)
    try:
        w = np.full((O, I), 0x38, np.uint8)
        for e in range(E):
            for p in range(2 if gated else 1):
                t.upload(e, w, np.full((1, 1), 1.0 if p else e + 1.0, np.float32), part=p)
                if e == 0:
                    one.upload(0, w, np.ones((1, 1), np.float32), part=p)
        q = torch.full((P, 128), 0x38, dtype=torch.uint8, device="cuda")
        at = torch.arange(P, device="cuda")
        s = (at % 7 + 1).float()
        cut = torch.sort(torch.randint(0, P + 1, (E + 1,), generator=torch.Generator().manual_seed(3)))[0].int().cuda()
        y = torch.full((P, O), 9.0, dtype=dtype, device="cuda")
        e = torch.searchsorted(cut.long(), at, right=True) - 1
        for row in (None, (P - 1 - at).int()):
            t.matmul_dev(ptr(q), ptr(s), P, ptr(row), ptr(cut), P, ptr(y), dtype=KIND[dtype], stream=stream())
            v = 5.0 * (s if row is None else s.flip(0))
            want = ((e + 1) * v * (v if gated else 1.0)).to(dtype)
            want = torch.where((e >= 0) & (e < E), want, 9.0)
            assert torch.equal(y, want[:, None].expand(P, O))
        S = 1 << 20
        one.matmul_ep_dev(ptr(q), ptr(s), S, ptr(y), dtype=KIND[dtype], stream=stream())
        v = 5.0 * s[:S]
        assert torch.equal(y[:S], (v * (v if gated else 1.0)).to(dtype)[:, None].expand(S, O))
    finally:
        t.close()
        one.close()


def test_experts_rows_alone():
    """A row's result does not depend on how many rows other experts have, nor on where it lies."""
    E, P, O, I = 6, 400, 90, 300
    c = Case(E, O, I, True, P, P, 5, res=False)
    try:
        def run(offs, row):
            y = torch.full((P, O), 9.0, device="cuda")
            D, r = torch.tensor(offs, dtype=torch.int32).cuda(), row.int().cuda()
            c.mat.matmul_dev(ptr(c.q), ptr(c.s), P, ptr(r), ptr(D), P, ptr(y), d_bias=ptr(c.b), act=1, stream=stream())
            return y

        a = run([0, 50, 100, 200, 200, 300, 400], torch.arange(P))
        row = torch.cat([torch.arange(40), torch.arange(100, 190), torch.arange(300, 400), torch.zeros(170, dtype=torch.long)])
        b = run([0, 40, 40, 130, 130, 130, 230], row)
        assert torch.equal(b[:40], a[:40]) and torch.equal(b[40:130], a[100:190]) and torch.equal(b[130:230], a[300:400])
        assert (b[230:] == 9.0).all()
    finally:
        c.mat.close()


def test_experts_wild_offsets():
    """Offsets that do not ascend or leave 0 .. P touch nothing outside y's P rows."""
    E, P, O, I = 70, 300, 40, 128
    c = Case(E, O, I, False, P, P, 5, res=False)
    try:
        for fill in (-5, 2 ** 31 - 1, -2 ** 31, P + 1):
            offs = torch.full((E + 1,), fill, dtype=torch.int32)
            offs[::3] = 100
            D = offs.cuda()
            y = torch.full((P + 64, O), 9.0, device="cuda")
            c.mat.matmul_dev(ptr(c.q), ptr(c.s), P, 0, ptr(D), P, y[32:].data_ptr(), stream=stream())
            torch.cuda.synchronize()
            assert (y[:32] == 9.0).all() and (y[32 + P:] == 9.0).all()
    finally:
        c.mat.close()


def test_experts_refusals_of_a_table():
    E, O, I = 3, 40, 200
    m, g = zz.Fp8Experts(E, O, I), zz.Fp8Experts(1, O, I, gated=True)
    try:
        q, s = torch.zeros(8, 256, dtype=torch.uint8, device="cuda"), torch.ones(2, 8, device="cuda")
        y = torch.full((9, O), 4.0, device="cuda")
        offs = torch.tensor([0, 2, 4, 8], dtype=torch.int32).cuda()
        row, b = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(2 * O, device="cuda")
        w, ws = np.zeros((O, I), np.uint8), np.ones((1, 2), np.float32)

        def experts(why, mat=m, **kw):
            a = dict(d_q=ptr(q), d_s=ptr(s), R=8, d_row=0, d_offs=ptr(offs), P=8, d_y=ptr(y), stream=stream())
            with pytest.raises(RuntimeError, match=why):
                mat.matmul_dev(**{**a, **kw})

        experts("without weights")
        for e in range(E):
            experts("without weights")
            m.upload(e, w, ws)
        m.matmul_dev(ptr(q), ptr(s), 8, 0, ptr(offs), 8, ptr(y), stream=stream())
        assert (y[:8] == 0.0).all()
        y.fill_(4.0)
        with pytest.raises(RuntimeError, match="no such"):
            m.upload(0, w, ws, part=1)
        for e in (-1, E):
            with pytest.raises(RuntimeError, match="no such"):
                m.upload(e, w, ws)
        experts("clamp", clamp=1.0)
        experts("closer", ldy=O - 1)
        experts("closer", d_res=ptr(b), ldr=O - 1)
        experts("overlaps", d_y=ptr(q))
        experts("overlaps", d_y=ptr(s))
        experts("overlaps", d_y=ptr(offs))
        experts("overlaps", d_y=ptr(row), d_row=ptr(row))
        experts("overlaps", d_y=ptr(b), d_bias=ptr(b))
        experts("overlaps", d_res=ptr(y) + 4 * O)
        experts("overlaps", d_res=ptr(y), ldr=O + 1)
        experts("2\\^32", R=1 << 24, d_row=ptr(row))
        L = zz.lib()
        for mat in (m, g):                       # the calls of one plain matrix do not take a table
            assert L.zz_fp8_upload(mat.id, w.ctypes.data_as(zz._u8p), ws.ctypes.data_as(zz._f32p)) == 0
            assert L.zz_fp8_matmul_dev(mat.id, ptr(q), ptr(s), 8, 0, ptr(y), 0, None) == 0 and "no such" in zz.last_error()
            assert L.zz_fp8_upload_dev(mat.id, ptr(q), ptr(s)) == 0
        assert L.zz_fp8_matmul_ep_dev(m.id, ptr(q), ptr(s), 8, None, 0, 0.0, None, 0, 0, ptr(y), 0, None) == 0
        g.upload(0, w, ws)
        assert L.zz_fp8_matmul_ep_dev(g.id, ptr(q), ptr(s), 8, None, 0, 0.0, None, 0, 0, ptr(y), 0, None) == 0
        assert "no weights" in zz.last_error()
        torch.cuda.synchronize()
        assert (y == 4.0).all()
    finally:
        m.close()
        g.close()


# ------------------------------------------------------------------ together
class Layer:
    """Experts of 8-bit floating point behind a routing: sorted, gate and up, rounded, down, back."""

    def __init__(self, S, K, E, D, MI, seed):
        self.S, self.K, self.E, self.D, self.MI = S, K, E, D, MI
        self.up, self.down = Case(E, MI, D, True, 1, 1, seed, BF16, bias=False, res=False), \
            Case(E, D, MI, False, 1, 1, seed + 50, F32, bias=False, res=False)
        n = S * K
        e = lambda *k, dtype=torch.int32: torch.zeros(*k, dtype=dtype, device="cuda")  # noqa: E731
        self.ids, self.w, self.x = e(S, K), e(S, K, dtype=F32), e(S, D, dtype=F32)
        self.offs, self.row, self.pos = e(E + 1), e(n), e(S, K)
        self.ws = e(zz.experts_ws_bytes(S, K, E), dtype=torch.uint8)
        self.q, self.s = e(S, zz.fp8_row_bytes(D), dtype=torch.uint8), e(R.blocks(D), S, dtype=F32)
        self.h, self.hq, self.hs = e(n, MI, dtype=BF16), e(n, zz.fp8_row_bytes(MI), dtype=torch.uint8), e(R.blocks(MI), n, dtype=F32)
        self.y, self.out = e(n, D, dtype=F32), e(S, D, dtype=F32)

    def __call__(self):
        st, n = stream(), self.S * self.K
        zz.experts_dispatch_dev(ptr(self.ids), self.S, self.K, self.E, ptr(self.offs), ptr(self.row), ptr(self.pos),
                                ptr(self.ws), self.ws.numel(), stream=st)
        zz.rows_fp8_dev(ptr(self.x), self.S, self.D, ptr(self.q), ptr(self.s), stream=st)
        self.up.mat.matmul_dev(ptr(self.q), ptr(self.s), self.S, ptr(self.row), ptr(self.offs), n, ptr(self.h), act=1,
                               dtype=zz.ZZ_BF16, stream=st)
        zz.rows_fp8_dev(ptr(self.h), n, self.MI, ptr(self.hq), ptr(self.hs), dtype=zz.ZZ_BF16, stream=st)
        self.down.mat.matmul_dev(ptr(self.hq), ptr(self.hs), n, 0, ptr(self.offs), n, ptr(self.y), stream=st)
        zz.experts_back_dev(ptr(self.y), ptr(self.pos), ptr(self.w), self.S, self.K, self.D, ptr(self.out), d_res=ptr(self.x), stream=st)

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.ids.copy_(routing(self.S, self.K, self.E, "dropped" if seed % 2 else "top", seed))
        w = torch.rand(self.S, self.K, generator=g)
        self.w.copy_(w / w.sum(1, keepdim=True))
        self.x.copy_(torch.randn(self.S, self.D, generator=g))

    def close(self):
        self.up.mat.close()
        self.down.mat.close()


@pytest.mark.parametrize("S, K, E, D, MI", [(1, 4, 16, 256, 96), (9, 3, 7, 300, 130), (300, 4, 16, 200, 64)])
def test_layer(S, K, E, D, MI):
    """The operators together, each stage against the definition on what the stage before gave."""
    L = Layer(S, K, E, D, MI, 3)
    try:
        for seed in (1, 2):
            print("case", S, seed, flush=True)
            L.fill(seed)
            L()
            torch.cuda.synchronize()
            o, r, p = X.sort(L.ids.cpu().numpy(), E)
            assert np.array_equal(L.offs.cpu(), o) and np.array_equal(L.pos.cpu(), p) and np.array_equal(L.row.cpu()[:r.size], r)
            v, sc = R.rows_exact(L.x.cpu().numpy())
            assert np.array_equal(R.e4m3_value(L.q.cpu().numpy()), v) and np.array_equal(L.s.cpu().numpy(), sc.astype(np.float32))
            L.up.xq, L.up.xs = L.q.cpu(), L.s.cpu()
            L.down.xq, L.down.xs = L.hq.cpu(), L.hs.cpu()
            for e in range(E):
                at = torch.arange(o[e], o[e + 1])
                if len(at):
                    near(L.h[at.cuda()], *L.up.want(e, torch.from_numpy(r)[at], at, 1, 0.0))
                    near(L.y[at.cuda()], *L.down.want(e, at, at, 0, 0.0))
            k = r.size
            v, sc = R.rows_exact(L.h[:k].float().cpu().numpy())
            assert np.array_equal(R.e4m3_value(L.hq[:k].cpu().numpy()), v)
            out, mag = X.back(L.y.cpu().numpy(), p, L.w.cpu().numpy(), L.x.cpu().numpy())
            assert np.all(np.abs(L.out.cpu().numpy() - out) <= X.back_bound(out, mag, K, R.HALF[F32]))
    finally:
        L.close()


def test_routed_by_a_layer():
    """The routing that zz_moe_forward_dev gives, as it is, through the sort and back."""
    import zzref as Z
    L = Z.make_layer("gemma", seed=5, E=16, D=512, MI=256, K=4)
    S = 70
    m = zz.MoeLayer(L.D, L.MI, L.E, L.K, L.gating, L.act, L.fmts, L.router, L.router_scale, L.pes, None, L.pre_ln, L.post_ln,
                    eps=L.eps)
    try:
        m.upload_all(L.experts)
        x = torch.from_numpy(Z.make_input(L, S, 5)).cuda()
        out, ids, w = torch.empty_like(x), torch.empty(S, L.K, dtype=torch.int32, device="cuda"), torch.empty(S, L.K, device="cuda")
        m.forward_dev(ptr(x), ptr(out), S, ptr(ids), ptr(w), stream())
        offs, row, pos, xs = dispatch(ids.cpu(), L.E, x, L.D)
        check_dispatch(ids.cpu(), L.E, (offs, row, pos, xs))
        d = m.debug(S)
        for u, lo, hi in zip(d["uniq"], d["offs"], d["offs"][1:]):   # the layer's own lists, expert by expert
            assert np.array_equal(row[offs[u]:offs[u + 1]].numpy(), d["rows"][lo:hi])
    finally:
        m.close()


def test_streams_and_graphs():
    """Two layers at once on two streams, and their captured graphs replayed with eager work
    between: every replay is the eager result."""
    for S in (2, 90, 2100):
        a, b, e = (Layer(S, 4, 16, 200, 64, 3) for _ in range(3))
        try:
            for L in (a, b, e):
                L.fill(1)
                L()
            torch.cuda.synchronize()
            graphs = []
            for L in (a, b):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    L()
                graphs.append(g)
            side = [torch.cuda.Stream(), torch.cuda.Stream()]
            for k in range(4):
                a.fill(10 + k)
                b.fill(20 + k)
                torch.cuda.synchronize()
                for L, g, st in zip((a, b), graphs, side):
                    with torch.cuda.stream(st):
                        g.replay() if k % 2 == 0 else L()
                torch.cuda.synchronize()
                for L in (a, b):
                    for t in ("ids", "w", "x"):
                        getattr(e, t).copy_(getattr(L, t))
                    e()
                    torch.cuda.synchronize()
                    n = int(e.offs[16])
                    assert torch.equal(L.out, e.out) and torch.equal(L.pos, e.pos) and torch.equal(L.row[:n], e.row[:n]), (S, k)
        finally:
            for L in (a, b, e):
                L.close()


def test_another_current_device_declines():
    """Where there is a second device; with one only, the device is the library's."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    with torch.cuda.device(1):
        with pytest.raises(RuntimeError, match="current"):
            zz.experts_back_dev(1 << 26, 1 << 27, 0, 4, 2, 8, 1 << 28)
