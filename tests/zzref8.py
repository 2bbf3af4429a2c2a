"""Plain 64-bit forms of the 8-bit rows, the fp8 product and the beam step (numpy and torch
on the CPU), with the bounds that the kernels' roundings allow."""
import numpy as np
import torch

U = 2.0 ** -24                   # half a step of f32, relative
BLK, FMAX, FLOOR = 128, 448.0, 2.0 ** -100
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def blocks(n):
    return -(-n // BLK)


def e4m3_half_step(v):
    """Half the distance between the e4m3 values around v (|v| <= 448)."""
    e = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -30)))
    return np.exp2(np.maximum(e, -6.0) - 4.0)


def e4m3_value(codes):
    """uint8 codes as float64, from the format's definition."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    return np.where((c & 127) == 127, np.nan, np.where(s == 1, -v, v))


def norm_rows(x, res, w, eps):
    """(h, y) in 64 bits; h is x + res as f32 holds it."""
    h = x.float()
    if res is not None:
        h = h + res.float()
    h = h.double().numpy()
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return h, h * r * (1.0 if w is None else w.double().numpy())


def check_rows(y, q, s, delta):
    """Codes q [S, whole blocks] and scales s [blocks, S] of rows y (64 bits), where the
    kernel's own y may be off by `delta`, relative: the scale by that and its division's
    rounding, a code by half a step beside what y / scale may be off."""
    S, D = y.shape
    nb = blocks(D)
    p = np.zeros((S, nb * BLK))
    p[:, :D] = y
    p = p.reshape(S, nb, BLK)
    want = np.maximum(np.abs(p).max(2), FLOOR) / FMAX
    s = s.double().numpy().T
    assert np.all(np.abs(s - want) <= (delta + U) * want)
    got = e4m3_value(q.numpy()).reshape(S, nb, BLK)
    assert not np.isnan(got).any()
    v = p / want[:, :, None]
    # y, its product with 448 / a, and that quotient's a and division
    off = np.abs(got - v)
    lim = e4m3_half_step(np.minimum(np.abs(v) * (1 + 2 * delta + 4 * U), FMAX)) + (2 * delta + 4 * U) * np.abs(v)
    assert np.all(off <= lim), (off - lim).max()
    assert not q.numpy()[:, D:].any()


def norm_delta(D):
    """How far a row's y may be off: the squares, their sum and the root are in 64 bits; the
    reciprocal's rounding to f32 and the two products are half a step each."""
    return 3 * U + D * 2.0 ** -52


def rows_exact(x):
    """(code values [S, whole blocks], scales [blocks, S]) of f32 rows, where nothing is open: the
    scale is f32's a / 448, a code the e4m3 value nearest to f32's x / scale, ties to even."""
    x = np.asarray(x, np.float32)
    S, D = x.shape
    p = np.zeros((S, blocks(D) * BLK), np.float32)
    p[:, :D] = x
    p = p.reshape(S, blocks(D), BLK)
    s = np.maximum(np.abs(p).max(2), np.float32(FLOOR)) / np.float32(FMAX)
    v = (p / s[:, :, None]).astype(np.float64)
    step = 2 * e4m3_half_step(v)
    return (np.round(v / step) * step).reshape(S, -1), s.T


def product(xq, xs, wq, ws, O, I):
    """(y, sum of |terms|) in 64 bits: rows' codes [S, whole blocks] (uint8), scales
    [blocks, S], codes [O, I], scales [blocks of O, blocks of I]."""
    x = e4m3_value(xq)[:, :I] * np.repeat(np.asarray(xs, np.float64).T, BLK, 1)[:, :I]
    w = e4m3_value(wq) * np.repeat(np.repeat(np.asarray(ws, np.float64), BLK, 0)[:O], BLK, 1)[:, :I]
    return x @ w.T, np.abs(x) @ np.abs(w).T


def product_bound(mag, want, I, dtype):
    """A block's 128 products are exact; each addition inside the matrix core may be off by a
    step (it need not round), each of the blocks' fma's and the joining additions by half a
    step, the scales' product by half a step; all of them relative to the terms' magnitudes;
    then the result's own rounding."""
    return (2 * BLK + blocks(I) + 16 + 2) * U * mag + HALF[dtype] * np.abs(want)


def beam_lists(logits, score, done, pad):
    """For N x W rows: each row's candidates in its own order (larger logit, lower token), as
    (tokens, totals in 64 bits)."""
    L = logits.double().numpy().copy()
    L[np.isnan(L)] = -np.inf
    L += 0.0
    c = np.asarray(score, np.float64).reshape(-1).copy()
    c[np.isnan(c)] = -np.inf
    rows = []
    for r in range(L.shape[0]):
        if done is not None and done.reshape(-1)[r]:
            rows.append((np.array([pad]), np.array([c[r]])))
            continue
        order = np.lexsort((np.arange(L.shape[1]), -L[r]))[:16]
        m = L[r].max()
        with np.errstate(invalid="ignore"):
            if m == -np.inf:
                t = np.full(L.shape[1], -np.inf)
            else:
                d = np.where(L[r] == m, 0.0, L[r] - m)
                t = c[r] + (d - np.log(np.exp(d).sum()))
        t = np.where(np.isnan(t), -np.inf, t)
        rows.append((order, t[order]))
    return rows


def beam_tol(V, total):
    """How far a total may be off: each of V exponentials by 2 U and its argument's two
    roundings (U |d| each, d = the logit's distance from the maximum, whose mean under the
    softmax is at most log V), a thread's chain of 64 additions and the waves' and chunks'
    few; and the score's rounding to f32."""
    return (2 * np.log(V) + 4 + 64 + 16) * U + U * abs(total)


def check_beam(logits, score, done, pad, eos, N, W, got):
    """The outputs of one step against the definition. Within a row the order is exact;
    between rows, beams whose totals differ by less than both are off may change places."""
    V = logits.shape[1]
    rows = beam_lists(logits, score, done, pad)
    so, par, tok, dn = (np.asarray(t) for t in got)
    for n in range(N):
        mine = rows[n * W:(n + 1) * W]
        cand = [(t, w, k) for w, (_, tt) in enumerate(mine) for k, t in enumerate(tt)]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        at = [0] * W
        for k in range(W):
            p, t = int(par[n, k]), int(tok[n, k])
            assert 0 <= p < W
            assert at[p] < len(mine[p][0]) and t == mine[p][0][at[p]], (n, k, p, t, at[p], mine[p][0][:4])
            total, want = mine[p][1][at[p]], cand[k][0]
            at[p] += 1
            if np.isinf(want) or np.isinf(total):
                assert total == want and so[n, k] == np.float32(want)
                if not any(np.isfinite(c[0]) for c in cand[k:]):
                    assert (p, t) == (cand[k][1], int(mine[cand[k][1]][0][cand[k][2]]))
            else:
                assert abs(total - want) <= 2 * beam_tol(V, want), (n, k, total, want)
                assert abs(float(so[n, k]) - total) <= beam_tol(V, total), (so[n, k], total)
                if all(abs(c[0] - want) > 2 * beam_tol(V, want) for c in cand if c[1] != cand[k][1]):
                    assert p == cand[k][1]
            fin = bool(done is not None and done.reshape(N, W)[n, p]) or (eos >= 0 and t == eos)
            assert bool(dn[n, k]) == fin
