"""Plain 64-bit forms of the sorting by expert, the way back, its gradient and the product's
epilogue (numpy on the CPU), with the bounds that the kernels' roundings allow."""
import numpy as np

import zzref8 as R

U = R.U


def sort(ids, E):
    """(offs [E + 1], row [kept], pos [S, K]) of ids [S, K], from the definition."""
    S, K = ids.shape
    flat = ids.reshape(-1).astype(np.int64)
    kept = np.nonzero((flat >= 0) & (flat < E))[0]
    order = kept[np.argsort(flat[kept], kind="stable")]
    pos = np.full(S * K, -1, np.int64)
    pos[order] = np.arange(order.size)
    offs = np.zeros(E + 1, np.int64)
    offs[1:] = np.cumsum(np.bincount(flat[kept], minlength=E)) if kept.size else 0
    return offs, order // K, pos.reshape(S, K)


def back(y, pos, w, res):
    """(out, sum of |terms|); pos outside y's rows is dropped, its weight unread."""
    S, K = pos.shape
    out = np.zeros((S, y.shape[1])) if res is None else res.astype(np.float64)
    mag = np.abs(out)
    for j in range(K):
        at = np.nonzero((pos[:, j] >= 0) & (pos[:, j] < S * K))[0]
        t = y[pos[at, j]].astype(np.float64) * (1.0 if w is None else w[at, j].astype(np.float64)[:, None])
        out[at] += t
        mag[at] += np.abs(t)
    return out, mag


def back_bound(out, mag, K, half):
    """K fma's of half a step each, relative to what has been added up; then the rounding."""
    off = (K + 1) * U * mag
    return off + half * (np.abs(out) + off)


def grad(dout, y, pos, w):
    """(dy by position as a dict of rows, dw, sum of |terms| of dw)"""
    S, K = pos.shape
    dy, dw, mag = {}, np.zeros((S, K)), np.zeros((S, K))
    g = dout.astype(np.float64)
    for s in range(S):
        for j in range(K):
            p = int(pos[s, j])
            if 0 <= p < S * K:
                dy[p] = g[s] * (1.0 if w is None else float(w[s, j]))
                if y is not None:
                    t = g[s] * y[p].astype(np.float64)
                    dw[s, j], mag[s, j] = t.sum(), np.abs(t).sum()
    return dy, dw, mag


def dw_bound(mag, D):
    """A lane's chain of up to 16 products, from 1025 columns on of 8 for each 2048, the wave's six
    and the waves' two joining additions."""
    return (max(16, 8 * -(-D // 2048)) + 9) * U * mag


def activated(v, act):
    """(act(v), how far the kernel's may be off for this very v): an exponential and a
    reciprocal of one unit in the last place (2 U), 1 + e and the last product half a step; the
    exponent's own roundings count by its size. gelu's: the cube's two products and its constant,
    the sum, the scale's constant (three factors, rounded twice) and product; silu's: the
    constant and the product. Below 2^-120 the reciprocal may be flushed."""
    if act == 0:
        return v, np.zeros_like(v)
    a = v if act == 2 else np.sqrt(8.0 / np.pi) * (v + 0.044715 * v ** 3)
    with np.errstate(over="ignore"):
        r = v / (1.0 + np.exp(-a))
    return r, (6 + (2 if act == 2 else 10) * np.minimum(np.abs(a), 200.0)) * U * np.abs(r) + 2.0 ** -110


def eights(xq, xs, wq, ws, O, I):
    """How far the 8-bit instructions' sums may be off beside their additions: within 8 columns each
    product is cut to 13 bits behind the leading one of the largest, so seven of the eight lose less
    than 2^-13 of it each (the largest itself has 8 bits). It is at most the product of the eights'
    largest codes."""
    S, nb = xq.shape[0], R.blocks(I)
    x, w = np.zeros((S, nb * R.BLK)), np.zeros((O, nb * R.BLK))
    x[:, :I], w[:, :I] = np.abs(R.e4m3_value(xq))[:, :I], np.abs(R.e4m3_value(wq))
    x = x.reshape(S, nb, 16, 8).max(3) * np.asarray(xs, np.float64).T[:, :, None]
    w = w.reshape(O, nb, 16, 8).max(3) * np.repeat(np.asarray(ws, np.float64), R.BLK, 0)[:O][:, :, None]
    return 7 * 2.0 ** -13 * (x.reshape(S, -1) @ w.reshape(O, -1).T)


def epilogue(sums, mags, I, bias, act, clamp, res, half, cut):
    """(y, bound): sums, mags and cut (what eights gives, or zeros) are lists of one or two [S, O]
    (gate, up) in 64 bits."""
    vs, ds = [], []
    for i, (v, m) in enumerate(zip(sums, mags)):
        d = (2 * R.BLK + R.blocks(I) + 16 + 2) * U * m + cut[i]     # as zzref8.product_bound
        if bias is not None:
            v = v + bias[i].astype(np.float64)
            d = d + U * (np.abs(v) + d)
        vs.append(v)
        ds.append(d)
    if len(vs) == 2 and clamp > 0:
        c = float(np.float32(clamp))
        vs = [np.minimum(vs[0], c), np.clip(vs[1], -c, c)]
    y, off = activated(vs[0], act)
    off = off + 1.2 * ds[0] * (1 + 40 * U)    # neither activation is steeper than 1.13
    if len(vs) == 2:
        off = off * np.abs(vs[1]) + np.abs(y) * ds[1] + off * ds[1]
        y = y * vs[1]
        # half a step, which below 2^-126, where f32's steps stop shrinking, is 2^-150: a product
        # of two sums of 1e-30 is 0
        off = off + U * (np.abs(y) + off) + 2.0 ** -149
    if res is not None:
        y = y + res.astype(np.float64)
        off = off + U * (np.abs(y) + off)
    return y, off + half * (np.abs(y) + off)
