"""Beam search's step, the reordering of states and a stack's search on the GPU."""
import numpy as np
import pytest
import torch

import zzref as Z
import zzref8 as R
import zunzuncito_amd as zz
from test_gpu_gemma import close_all, gpu_block

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
KIND = {F32: zz.ZZ_F32, BF16: zz.ZZ_BF16}


@pytest.fixture(autouse=True, scope="module")
def _up():
    zz.init()


def stream():
    return torch.cuda.current_stream().cuda_stream


def step(logits, score, done, N, W, V, eos=1, pad=0, ldl=0, off=0, alias=False):
    """One step; outputs [N, W] on the host, and the guards behind them looked at."""
    dt = logits.dtype
    buf = logits.cuda()
    sc = score.cuda()
    dn = None if done is None else done.to(torch.uint8).cuda()
    n = N * W
    so = sc if alias else torch.full((n + 2,), -9.0, device="cuda")
    pa = torch.full((n + 2,), -9, dtype=torch.int32, device="cuda")
    tk = torch.full((n + 2,), -9, dtype=torch.int32, device="cuda")
    do = dn if alias and dn is not None else torch.full((n + 2,), 77, dtype=torch.uint8, device="cuda")
    need = zz.beam_ws_bytes(N, W, V)
    ws = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    zz.beam_step_dev(buf.data_ptr() + off * buf.element_size(), N, W, V, sc.data_ptr(), so.data_ptr(), pa.data_ptr(),
                     tk.data_ptr(), ws.data_ptr(), need, d_done=0 if dn is None else dn.data_ptr(),
                     d_done_out=do.data_ptr(), eos=eos, pad=pad, dtype=KIND[dt], ldl=ldl, stream=stream())
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xAB).all()) and bool((pa[n:] == -9).all()) and bool((tk[n:] == -9).all())
    if not alias:
        assert bool((so[n:] == -9.0).all()) and bool((do[n:] == 77).all())
    return [t.view(-1)[:n].view(N, W).cpu() for t in (so, pa, tk, do)]


def check(logits, score, done, N, W, V, eos=1, pad=0, view=None, **kw):
    got = step(logits, score, done, N, W, V, eos, pad, **kw)
    R.check_beam(logits if view is None else view, score, done, pad, eos, N, W, got)
    return got


def draw(N, W, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (3 * torch.randn(N * W, V, generator=g)).to(dtype), -3 - 5 * torch.rand(N, W, generator=g), g


# one token, fewer tokens than beams, sizes around a thread's, a wave's and a chunk's share,
# row starts that no 16-byte line holds, the widest search, the two-piece and eight-piece forms
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, W, V", [(1, 1, 1), (1, 4, 1), (2, 3, 2), (1, 16, 5), (3, 5, 17), (1, 4, 1000), (2, 16, 2047),
                                     (1, 2, 2048), (1, 2, 2049), (2, 7, 8191), (1, 3, 8193), (5, 4, 32768), (1, 16, 100003),
                                     (40, 13, 5000), (1, 1, 262144), (2, 8, 262143), (1, 2, zz.ZZ_BEAM_MAXV)])
def test_step(dtype, N, W, V):
    print("case", N, W, V, dtype, flush=True)
    logits, score, g = draw(N, W, V, dtype, N + W + V)
    check(logits, score, None, N, W, V)
    if N * W > 1:
        done = torch.rand(N, W, generator=g) < 0.4
        check(logits, score, done, N, W, V, pad=V - 1)
        first = torch.full((N, W), -float("inf"))
        first[:, 0] = 0.0
        got = check(logits, first, None, N, W, V)
        if V >= W:
            assert bool((got[1] == 0).all())


# both sides of the vocabulary that one launch takes; a last chunk of a few tokens; lists for
# one wave's lanes and for more; one beam, one chunk or one token of each beam ahead of the rest
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, W, V", [(9, 16, 2048), (9, 16, 2049), (2, 5, 2060), (3, 16, 6147), (1, 9, 8200), (2, 16, 20000),
                                     (70, 8, 16400), (1, 4, 65540)])
@pytest.mark.parametrize("ahead", ["beam", "chunk", "tokens", "few"])
def test_step_places(dtype, N, W, V, ahead):
    logits, score, g = draw(N, W, V, dtype, N + V)
    if ahead == "beam":
        score[:, W // 2] = 100.0
    elif ahead == "chunk":
        logits[:, -(V % 2048 or 2048):] += 20.0
    elif ahead == "tokens":
        score[:] = -1.0
        logits[:] = logits[:1]                           # equal beams: every total W times
    else:
        keep = torch.rand(N * W, V, generator=g) < 3 * W / V
        keep[:, V // 2] = True
        logits[~keep] = -float("inf")
    check(logits, score, None, N, W, V)
    done = torch.rand(N, W, generator=g) < 0.5
    check(logits, score, done, N, W, V)


def test_step_widest():
    """The most beams over the largest vocabulary: the longest lists that a merge holds."""
    N, W, V = 1, 16, zz.ZZ_BEAM_MAXV
    logits, score, _ = draw(N, W, V, F32, 4)
    check(logits, score, None, N, W, V)


def test_step_and_reorder_past_32_bits():
    """Logits and states at offsets that 32 bits do not hold: some sequences of many, against
    64 bits and against the rows moved one by one."""
    N, W, V = 1200, 16, 131072
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.empty(N * W, V, dtype=BF16, device="cuda").normal_(generator=g)
    score = -torch.rand(N, W, device="cuda", generator=g)
    so, pa, tk = torch.empty_like(score), *(torch.empty(N, W, dtype=torch.int32, device="cuda") for _ in range(2))
    do = torch.empty(N, W, dtype=torch.uint8, device="cuda")
    ws = torch.empty(zz.beam_ws_bytes(N, W, V), dtype=torch.uint8, device="cuda")
    zz.beam_step_dev(logits.data_ptr(), N, W, V, score.data_ptr(), so.data_ptr(), pa.data_ptr(), tk.data_ptr(), ws.data_ptr(),
                     ws.numel(), d_done_out=do.data_ptr(), eos=1, dtype=zz.ZZ_BF16, stream=stream())
    torch.cuda.synchronize()
    for n in (0, N // 2, N - 1):
        got = [t[n:n + 1].cpu() for t in (so, pa, tk, do)]
        R.check_beam(logits[n * W:(n + 1) * W].cpu(), score[n:n + 1].cpu(), None, 0, 1, 1, W, got)
    states = logits.view(N, W, V)                        # as states of 256 KB a beam, in place
    keep = states[:, :, ::4099].clone()
    zz.beam_reorder_dev(logits.data_ptr(), logits.data_ptr(), pa.data_ptr(), N, W, row_stride=2 * V, row_bytes=2 * V - 6,
                        stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(states[:, :, ::4099], torch.gather(keep, 1, pa.long()[:, :, None].expand_as(keep)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V, ldl, off", [(1001, 1001, 1), (1001, 1010, 3), (9000, 9001, 0), (4096, 8192, 4)])
def test_step_strides(dtype, V, ldl, off):
    N, W = 2, 4
    g = torch.Generator().manual_seed(V)
    buf = (2 * torch.randn(N * W * ldl + off, generator=g)).to(dtype)
    buf[:off] = 1000.0                                   # never to be seen
    rows = buf[off:].view(N * W, ldl)
    rows[:, V:] = 1000.0
    score = -torch.rand(N, W, generator=g)
    check(buf, score, None, N, W, V, view=rows[:, :V], ldl=ldl, off=off)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 40000])
def test_step_ties(dtype, V):
    """Equal logits everywhere, in runs across threads', waves' and chunks' shares, minus zero
    beside zero, and equal beams: the lower beam and the lower token first."""
    N, W = 1, 8
    same = torch.zeros(W, V)
    same[:, 1::2] = -0.0
    score = torch.zeros(N, W)
    got = check(same.to(dtype), score, None, N, W, V)
    assert torch.equal(got[1][0], torch.zeros(W, dtype=torch.int32))
    assert torch.equal(got[2][0], torch.arange(W, dtype=torch.int32))
    runs = torch.zeros(W, V)
    runs[:, V // 3:V // 3 + 100] = 5.0
    runs[:, -3:] = 5.0
    got = check(runs.to(dtype), score, None, N, W, V)
    assert torch.equal(got[2][0], torch.arange(V // 3, V // 3 + W, dtype=torch.int32))
    few = torch.full((W, V), -2.0)
    few[:, [3, V // 2, V - 1]] = 1.0                     # three a beam: two beams and two of the third
    got = check(few.to(dtype), score, None, N, W, V)
    assert got[1][0].tolist() == [0, 0, 0, 1, 1, 1, 2, 2]
    assert got[2][0].tolist() == [3, V // 2, V - 1, 3, V // 2, V - 1, 3, V // 2]
    one = torch.full((W, V), -30.0)
    one[:, V - 2] = 9.0
    one[:, 5] = 9.0
    check(one.to(dtype), torch.tensor([[-1.0, -2, -1, -3, -1, -2, -9, -1]]), None, N, W, V)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [50, 9000])
def test_step_masks(dtype, V):
    """Rows whose mask leaves one, a few or nothing; NaN, infinities and the type's lowest
    value in masked places; beams at minus infinity, at NaN, finished."""
    N, W = 2, 6
    inf = float("inf")
    logits, score, g = draw(N, W, V, dtype, V)
    L = logits.float()
    L[0, :] = -inf                                       # nothing left
    L[1, :] = -inf
    L[1, V - 1] = 2.0                                    # one
    L[2, :] = torch.finfo(dtype).min
    L[2, 7:9] = 0.5
    L[3, ::2] = float("nan")
    L[4, 3], L[4, V - 4] = inf, inf                      # shares its probability
    L[5, :] = float("nan")
    L[7, :] = -inf
    L[8, :] = torch.finfo(dtype).min                     # all at the lowest value: uniform
    L = L.to(dtype)
    check(L, score, None, N, W, V)
    score[0, 2], score[1, 3] = -inf, float("nan")
    check(L, score, None, N, W, V)
    done = torch.zeros(N, W, dtype=torch.bool)
    done[0, 1], done[1] = True, True                     # a whole sequence finished
    got = check(L, score, done, N, W, V, eos=7, pad=7)
    assert bool((got[2][1] == 7).all()) and bool((got[3][1] == 1).all())
    none = torch.full((N * W, V), -inf).to(dtype)
    got = check(none, score, None, N, W, V)              # W candidates all the same
    assert bool(torch.isinf(got[0]).all())
    check(none, torch.full((N, W), -inf), done, N, W, V)


def test_step_in_place_and_no_flags():
    N, W, V = 3, 5, 3001
    logits, score, g = draw(N, W, V, F32, 9)
    done = torch.rand(N, W, generator=g) < 0.3
    plain = step(logits, score, done, N, W, V)
    over = step(logits, score, done, N, W, V, alias=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, over))
    no = step(logits, score, done, N, W, V, eos=-1)
    assert torch.equal(no[3].bool(), done.gather(1, no[1].long()))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, F32])
@pytest.mark.parametrize("N, W, outer, cap, used, width", [(1, 1, 1, 1, 1, 1), (1, 4, 2, 8, 5, 32), (3, 5, 1, 7, 7, 33),
                                                           (2, 16, 3, 64, 33, 8), (7, 8, 2, 300, 257, 24), (2, 3, 2, 5, 1, 7)])
def test_reorder(dtype, N, W, outer, cap, used, width):
    g = torch.Generator().manual_seed(N * W)
    src = (100 * torch.randn(outer, N * W, cap, width, generator=g)).to(dtype)
    for kind in ("random", "same", "one"):
        par = torch.randint(0, W, (N, W), generator=g, dtype=torch.int32)
        if kind == "same":
            par = torch.arange(W, dtype=torch.int32).repeat(N, 1)
        elif kind == "one":
            par[:] = W - 1
        at = (torch.arange(N)[:, None] * W + par.long()).view(-1)
        P = par.cuda()
        esz = src.element_size()
        row = cap * width * esz
        for inplace in (False, True):
            S = src.cuda()
            D = S if inplace else torch.full_like(S, 3)
            want = D.cpu().clone()
            want[:, :, :used] = src[:, at][:, :, :used]
            zz.beam_reorder_dev(D.data_ptr(), S.data_ptr(), P.data_ptr(), N, W, outer, N * W * row, row,
                                used * width * esz, stream())
            assert torch.equal(D.cpu(), want), (kind, inplace)
            if not inplace:
                assert torch.equal(S.cpu(), src)


def test_reorder_bad_parents_and_offsets():
    """A parent outside the beams keeps the row; starts and strides of every alignment; planes
    further apart than their rows."""
    N, W = 2, 4
    g = torch.Generator().manual_seed(3)
    par = torch.tensor([[-1, 0, 4, 1 << 30], [3, 3, -(1 << 31), 0]], dtype=torch.int32)
    good = torch.where((par < 0) | (par >= W), torch.arange(W, dtype=torch.int32), par)
    at = (torch.arange(N)[:, None] * W + good.long()).view(-1)
    P = par.cuda()
    for off, row, used in ((0, 64, 64), (1, 50, 49), (4, 52, 50), (8, 48, 33), (16, 48, 1), (3, 7, 7)):
        plane = N * W * row + 16
        src = torch.randint(0, 255, (off + 2 * plane,), generator=g, dtype=torch.uint8)
        for inplace in (False, True):
            S = src.cuda()
            D = S if inplace else torch.full_like(S, 9)
            want = D.cpu().clone()
            for o in range(2):
                a = src[off + o * plane:][:N * W * row].view(N * W, row)
                want[off + o * plane:][:N * W * row].view(N * W, row)[:, :used] = a[at][:, :used]
            zz.beam_reorder_dev(D.data_ptr() + off, S.data_ptr() + off, P.data_ptr(), N, W, 2, plane, row, used, stream())
            assert torch.equal(D.cpu(), want), (off, row, used, inplace)


def test_captured_search():
    """Two captured steps with a workspace each, replayed on two streams with eager work
    between: each replay is the eager result."""
    N, W, V = 2, 4, 5000
    g = torch.Generator(device="cuda").manual_seed(2)

    class Run:
        def __init__(self):
            self.L = torch.zeros(N * W, V, device="cuda")
            self.sc = torch.zeros(N, W, device="cuda")
            self.so = torch.zeros(N, W, device="cuda")
            self.pa, self.tk = (torch.zeros(N, W, dtype=torch.int32, device="cuda") for _ in range(2))
            self.ws = torch.empty(zz.beam_ws_bytes(N, W, V), dtype=torch.uint8, device="cuda")
            self.src = torch.zeros(3, N * W, 40, device="cuda")
            self.dst = torch.zeros(3, N * W, 40, device="cuda")

        def __call__(self):
            zz.beam_step_dev(self.L.data_ptr(), N, W, V, self.sc.data_ptr(), self.so.data_ptr(), self.pa.data_ptr(),
                             self.tk.data_ptr(), self.ws.data_ptr(), self.ws.numel(), stream=stream())
            zz.beam_reorder_dev(self.dst.data_ptr(), self.src.data_ptr(), self.pa.data_ptr(), N, W, 3, N * W * 160, 160,
                                160, stream())

        def out(self):
            return [t.clone() for t in (self.so, self.pa, self.tk, self.dst)]

    one, two, eager = Run(), Run(), Run()
    torch.cuda.synchronize()
    graphs = []
    for r in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r()
        graphs.append(gr)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for r in (one, two):
            r.L.normal_(generator=g)
            r.sc.normal_(generator=g)
            r.src.normal_(generator=g)
        torch.cuda.synchronize()
        for st, gr in zip(side, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for r in (one, two):
            for n in ("L", "sc", "src"):
                getattr(eager, n).copy_(getattr(r, n))
            eager()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager.out(), r.out())), k


def test_norm_product_beam_together():
    """A head in 8-bit floating point under a search: residual and norm, the product over the
    vocabulary, the step, the reordering of a cache and of the rows themselves."""
    N, W, D, V = 2, 3, 320, 1000
    g = torch.Generator().manual_seed(12)
    x, res = torch.randn(N * W, D, generator=g), torch.randn(N * W, D, generator=g)
    w = 1 + 0.1 * torch.randn(D, generator=g)
    r = np.random.default_rng(12)
    wq = np.where(((c := r.integers(0, 256, (V, D)).astype(np.uint8)) & 127) == 127, 3, c).astype(np.uint8)
    ws = np.exp(r.normal(-9.5, 0.2, (R.blocks(V), R.blocks(D)))).astype(np.float32)
    score = -torch.rand(N, W, generator=g)
    cache = torch.randn(2, N * W, 10, 16, generator=g)
    m = zz.Fp8Matrix(V, D)
    try:
        m.upload(wq, ws)
        X, Rs, Wt, Sc, Ca = (t.cuda() for t in (x, res, w, score, cache))
        q = torch.empty(N * W, 384, dtype=torch.uint8, device="cuda")
        s = torch.empty(3, N * W, device="cuda")
        y = torch.empty(N * W, V, device="cuda")
        pa, tk = (torch.empty(N, W, dtype=torch.int32, device="cuda") for _ in range(2))
        wsb = torch.empty(zz.beam_ws_bytes(N, W, V), dtype=torch.uint8, device="cuda")
        st = stream()
        zz.add_norm_fp8_dev(X.data_ptr(), Rs.data_ptr(), Rs.data_ptr(), Wt.data_ptr(), N * W, D, 1e-6, q.data_ptr(),
                            s.data_ptr(), stream=st)
        m.matmul_dev(q.data_ptr(), s.data_ptr(), N * W, y.data_ptr(), stream=st)
        dn = torch.zeros(N, W, dtype=torch.uint8, device="cuda")
        zz.beam_step_dev(y.data_ptr(), N, W, V, Sc.data_ptr(), Sc.data_ptr(), pa.data_ptr(), tk.data_ptr(), wsb.data_ptr(),
                         wsb.numel(), d_done=dn.data_ptr(), d_done_out=dn.data_ptr(), eos=2, stream=st)
        zz.beam_reorder_dev(Ca.data_ptr(), Ca.data_ptr(), pa.data_ptr(), N, W, 2, N * W * 640, 640, 320, st)
        zz.beam_reorder_dev(Rs.data_ptr(), Rs.data_ptr(), pa.data_ptr(), N, W, 1, 0, 4 * D, 4 * D, st)
        torch.cuda.synchronize()
        h, yn = R.norm_rows(x, res, w, float(np.float32(1e-6)))
        R.check_rows(yn, q.cpu(), s.cpu(), R.norm_delta(D))
        want, mag = R.product(q.cpu().numpy(), s.cpu().numpy(), wq, ws, V, D)
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= R.product_bound(mag, want, D, F32))
        R.check_beam(y.cpu(), score, None, 0, 2, N, W, [t.cpu() for t in (Sc, pa, tk, dn)])
        at = (torch.arange(N)[:, None] * W + pa.cpu().long()).view(-1)
        ref = cache.clone()
        ref[:, :, :5] = cache[:, at][:, :, :5]
        assert torch.equal(Ca.cpu(), ref) and torch.equal(Rs.cpu(), (x + res)[at])
    finally:
        m.close()


def tied_head(V, D, seed):
    r = np.random.default_rng(seed)
    d = r.normal(0.0, 0.004, (V * D // 32, 1)).astype(np.float16)
    q = r.integers(0, 256, (V * D // 32, 16)).astype(np.uint8)
    return np.concatenate([d.view(np.uint8).reshape(-1, 2), q], 1).reshape(-1)


@pytest.mark.parametrize("W, eos, flash", [(1, -1, False), (3, 9, False), (5, -1, False), (16, 3, False), (4, 2, True)])
def test_stack_search(W, eos, flash):
    """zz_stack_beam_dev step by step: the same embedding, blocks, head and step called one by
    one; one beam is the greedy decode. With a FlashHead only the probed tokens have logits."""
    L = Z.make_layer("gemma", seed=39, E=16, K=4, D=512, MI=256)
    b, m, d = gpu_block(L, Z.make_dense(L.D, 512, 40))
    V, D, n = 1024, L.D, 6
    head = zz.Head(tied_head(V, D, 4), V, D, np.ones(D, np.float32), 1e-6, float(np.sqrt(D)), 30.0)
    stack = zz.Stack([b], head)
    try:
        if flash:
            ids = np.random.default_rng(8).permutation(V).astype(np.int32).reshape(32, 32)
            head.flash(tied_head(32, D, 5), 32, ids, 32, 5, np.ones(32, np.float32), 1, np.array([2, 7], np.int32))
            head.use_flash(True)
        start = torch.tensor([17], dtype=torch.int32, device="cuda")
        seq = torch.full((W + 1, n + 1), -5, dtype=torch.int32, device="cuda")
        score = torch.full((W + 1,), -5.0, device="cuda")
        for _ in range(2):                               # the second call finds its rows there
            stack.beam_dev(start.data_ptr(), W, n, seq.data_ptr(), score.data_ptr(), eos=eos, stream=stream())
        torch.cuda.synchronize()
        assert bool((seq[W] == -5).all()) and float(score[W]) == -5.0
        hist = [[17] for _ in range(W)]
        sc = torch.full((1, W), -float("inf"))
        sc[0, 0] = 0.0
        dn = torch.zeros(1, W, dtype=torch.bool)
        for i in range(n):
            H = torch.from_numpy(head.embed(np.array([t[-1] for t in hist], np.int32))).cuda()
            stack.prefill_dev(H.data_ptr(), W, 0, stream())
            lg = torch.empty(W, V, device="cuda")
            for w in range(0, W, 4):
                k = min(4, W - w)
                head.logits_dev(H[w:].data_ptr(), k, lg[w:].data_ptr(), stream=stream())
            torch.cuda.synchronize()
            assert flash == bool(torch.isinf(lg).any())
            so, pa, tk, do = check(lg.cpu(), sc, dn, 1, W, V, eos=eos, pad=max(eos, 0))
            hist = [hist[int(p)] + [int(t)] for p, t in zip(pa[0], tk[0])]
            sc, dn = so, do.bool()
        assert seq[:W].cpu().tolist() == hist
        assert torch.equal(score[:W].cpu(), sc[0])
        if W == 1:
            tok = torch.tensor([17] + [0] * n, dtype=torch.int32, device="cuda")
            stack.decode_dev(tok.data_ptr(), n, stream=stream())
            assert tok.cpu().tolist() == hist[0]
        stack.beam_dev(start.data_ptr(), W, 0, seq.data_ptr(), score.data_ptr(), eos=eos, stream=stream())
        torch.cuda.synchronize()
        assert seq.view(-1)[:W].cpu().tolist() == [17] * W
        with pytest.raises(RuntimeError, match="W <= 16"):
            stack.beam_dev(start.data_ptr(), 17, n, seq.data_ptr(), score.data_ptr(), stream=stream())
        with pytest.raises(RuntimeError, match="overlaps"):
            stack.beam_dev(seq.data_ptr() + 4 * n, W, n, seq.data_ptr(), score.data_ptr(), stream=stream())
    finally:
        stack.close()
        head.close()
        close_all(b, m, d)


@pytest.mark.parametrize("gone", ["block", "head"])
def test_stack_search_declined(gone):
    """A search that is declined on its way, because a block or the head is no longer there,
    leaves the outputs as they were; longer and wider searches follow shorter ones."""
    L = Z.make_layer("gemma", seed=41, E=16, K=4, D=512, MI=256)
    b, m, d = gpu_block(L, Z.make_dense(L.D, 512, 40))
    V, D = 1024, L.D
    head = zz.Head(tied_head(V, D, 4), V, D, np.ones(D, np.float32), 1e-6, float(np.sqrt(D)), 30.0)
    stack = zz.Stack([b], head)
    try:
        start = torch.tensor([17], dtype=torch.int32, device="cuda")

        def search(W, n):
            seq = torch.full((W, n + 1), -5, dtype=torch.int32, device="cuda")
            score = torch.full((W,), -5.0, device="cuda")
            try:
                stack.beam_dev(start.data_ptr(), W, n, seq.data_ptr(), score.data_ptr(), stream=stream())
                torch.cuda.synchronize()
                return seq.cpu(), score.cpu(), None
            except RuntimeError as e:
                torch.cuda.synchronize()
                return seq.cpu(), score.cpu(), str(e)

        short, long = search(3, 2), search(3, 300)
        assert short[2] is None and long[2] is None and bool((long[0] >= 0).all())
        again = search(3, 2)
        assert torch.equal(again[0], short[0]) and torch.equal(again[1], short[1])
        (b if gone == "block" else head).close()
        seq, score, why = search(3, 2)
        assert why and ("gone" if gone == "block" else "zz_head") in why
        assert bool((seq == -5).all()) and bool((score == -5.0).all())
    finally:
        stack.close()
        head.close()
        close_all(b, m, d)


@pytest.mark.parametrize("N, W, row", [(5, 3, 1 << 23), (2, 4, 9000001), (3, 8, 1 << 22), (1, 16, 5000013)])
def test_reorder_past_the_caches(N, W, row):
    """States of 64 MiB and more, for each number of rows that a thread holds, in place and not,
    with bytes behind the last whole piece and with none."""
    g = torch.Generator(device="cuda").manual_seed(W)
    src = torch.randint(0, 255, (N, W, row), generator=g, dtype=torch.uint8, device="cuda")
    par = torch.randint(0, W, (N, W), generator=g, dtype=torch.int32, device="cuda")
    used = row - 1 if row % 2 else row
    assert N * W * used >= 64 << 20
    want = torch.stack([src[n, par[n].long(), :used] for n in range(N)])
    dst = torch.full_like(src, 3)
    for to in (dst, src):
        last = to[:, :, used:].clone()
        zz.beam_reorder_dev(to.data_ptr(), src.data_ptr(), par.data_ptr(), N, W, row_stride=row, row_bytes=used, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(to[:, :, :used], want) and torch.equal(to[:, :, used:], last)
