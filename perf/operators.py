"""The 8-bit rows, the fp8 product and the beam step, measured against their plain forms.

What a decoder does around its large tables: the residual's addition, the root mean square
norm and the rounding to e4m3 codes with a scale for each 128 values (kind "norm", and
"rows" where activations are only rounded); the product of such rows with e4m3 weights that
have a scale for each 128 x 128 block (kind "product"); and one step of beam search over
the logits with the reordering of the beams' states (kind "beam").

Hidden, intermediate and vocabulary sizes are those of this repository's layers and tests
(2816, 2112 and 4224 = 2 x 2112, 2048, 704, 1088, 262144), and generic ones.
"""
import math

import torch

own = False

EPS = 1e-6
BLK = 128
FMAX = 448.0                     # the largest e4m3 value
FLOOR = 2.0 ** -100              # a block's largest magnitude counts as at least this
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token between two layers: a launch and a row's latency
        dict(name="norm_decode_1", kind="norm", tokens=1, width=2816, dtype="f32", wide=1),
        # a serving batch with activations in 16 bits
        dict(name="norm_batch_37", kind="norm", tokens=37, width=2048, dtype="bf16", wide=1),
        # the second half of a gate|up buffer rounded for the down product: rows apart by
        # twice their width, 16 blocks and a half
        dict(name="rows_prefill_1500", kind="rows", tokens=1500, width=2112, dtype="bf16", wide=2),
        # a long prompt's rows, in 32 bits
        dict(name="norm_prefill_8192", kind="norm", tokens=8192, width=2816, dtype="f32", wide=1),
        # one token through a down projection: the weights' bytes and latency
        dict(name="product_decode_1", kind="product", tokens=1, rows=2816, cols=2112, dtype="f32"),
        # a ragged serving batch on a matrix that no tile divides
        dict(name="product_batch_21", kind="product", tokens=21, rows=1000, cols=1088, dtype="bf16"),
        # three sequences against a whole vocabulary: the weights' bytes alone
        dict(name="product_head_3", kind="product", tokens=3, rows=262144, cols=2816, dtype="f32"),
        # an ordinary prefill chunk through gate|up
        dict(name="product_prefill_512", kind="product", tokens=512, rows=4224, cols=2816, dtype="f32"),
        # a long prompt through the same: the matrix cores
        dict(name="product_prefill_8192", kind="product", tokens=8192, rows=4224, cols=2816, dtype="bf16"),
        # the first step of one search: one live beam, the others at minus infinity
        dict(name="beam_first_1", kind="beam", seqs=1, beams=4, vocab=32768, dtype="f32", first=True,
             probed=1.0, done=0, layers=2, cap=64, len=33, width=128),
        # several users, five beams, logits in 16 bits (many equal ones), a third finished
        dict(name="beam_batch_7", kind="beam", seqs=7, beams=5, vocab=100003, dtype="bf16", first=False,
             probed=1.0, done=3, layers=4, cap=256, len=177, width=200),
        # a full batch under the whole vocabulary, long states
        dict(name="beam_batch_16", kind="beam", seqs=16, beams=8, vocab=262144, dtype="f32", first=False,
             probed=1.0, done=0, layers=4, cap=1024, len=1000, width=256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "rows", "product", "product", "product", "head", "beam", "beam"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("norm", "rows"):
        width = _log_int(rng, 64, 8192)
        tokens = _log_int(rng, 1, min(16384, 8192 * 2816 // width))
        return dict(kind=kind, tokens=tokens, width=width, dtype=dtype, wide=rng.choice([1, 1, 2]))
    if kind == "head":
        return dict(kind="product", tokens=rng.randint(1, 4), rows=_log_int(rng, 8192, 262144),
                    cols=_log_int(rng, 512, 2816), dtype=dtype)
    if kind == "product":
        rows, cols = _log_int(rng, 64, 8448), _log_int(rng, 64, 8192)
        tokens = _log_int(rng, 1, min(8192, 8192 * 4224 * 2816 // (rows * cols)))
        return dict(kind=kind, tokens=tokens, rows=rows, cols=cols, dtype=dtype)
    beams = rng.randint(1, 16)
    return dict(kind=kind, seqs=_log_int(rng, 1, 128 // beams), beams=beams, vocab=_log_int(rng, 1000, 262144),
                dtype=dtype, first=rng.random() < 0.2, probed=rng.choice([1.0, 1.0, 0.1]),
                done=rng.choice([0, 0, 2, 5]), layers=rng.randint(1, 4), cap=1024, len=_log_int(rng, 1, 1000),
                width=rng.randint(16, 256))


# ------------------------------------------------------------------ inputs
class State:
    """What a program holds between calls; a weight handle is given back with it."""
    handle = None

    def __del__(self):
        if self.handle is not None:
            self.handle.close()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(case, seed):
    """x and the residual [S, wide * D] (a row's first D values are used) and the norm's
    weight: a residual stream's values, some columns far larger than the rest."""
    g = _gen(seed)
    S, D, t = case["tokens"], case["width"], TYPES[case["dtype"]]
    wide = case["wide"] * D
    col = 1 + 9 * (torch.rand(wide, generator=g, device="cuda") < 0.01)
    x = (torch.randn(S, wide, generator=g, device="cuda") * col).to(t)
    res = (3 * torch.randn(S, wide, generator=g, device="cuda") * col).to(t)
    w = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
    return x, res, w


def _ceil(n):
    return -(-n // BLK)


def _coded(v, br):
    """e4m3 codes of a matrix and the f32 scales of its br x 128 blocks."""
    O, I = v.shape
    p = torch.nn.functional.pad(v, (0, _ceil(I) * BLK - I, 0, -(-O // br) * br - O))
    b = p.view(p.shape[0] // br, br, _ceil(I), BLK)
    s = b.abs().amax((1, 3)).clamp_min(FLOOR) / FMAX
    q = (b / s[:, None, :, None]).view(p.shape).to(torch.float8_e4m3fn)
    return q[:O], s


def _product_inputs(case, seed):
    """Weights [O, I] as codes and block scales, and activation rows as codes [S, I up to
    whole blocks] and scales [blocks, S]."""
    g = _gen(seed)
    S, O, I = case["tokens"], case["rows"], case["cols"]
    wq, ws = _coded(torch.empty(O, I, device="cuda").normal_(0.0, 0.02, generator=g), BLK)
    col = 1 + 9 * (torch.rand(I, generator=g, device="cuda") < 0.01)
    xq, xs = _coded(torch.randn(S, I, generator=g, device="cuda") * col, 1)
    return wq[:, :I].contiguous(), ws, xq.contiguous(), xs.t().contiguous()


def _beam_inputs(case, seed):
    g = _gen(seed)
    N, W, V, t = case["seqs"], case["beams"], case["vocab"], TYPES[case["dtype"]]
    logits = 3 * torch.randn(N * W, V, generator=g, device="cuda")
    if case["probed"] < 1.0:     # a head that scores only the likely part of its vocabulary
        logits.masked_fill_(torch.rand(N * W, V, generator=g, device="cuda") >= case["probed"], -math.inf)
    score = -4.0 - 6.0 * torch.rand(N, W, generator=g, device="cuda")
    if case["first"]:
        score[:] = -math.inf
        score[:, 0] = 0.0
    done = torch.zeros(N, W, dtype=torch.bool, device="cuda")
    if case["done"] and not case["first"]:
        done.view(-1)[seed % case["done"]::case["done"]] = True
    states = torch.randn(case["layers"], N * W, case["cap"], case["width"], generator=g, device="cuda")
    return logits.to(t), score, done, states.to(torch.bfloat16)


def prepare(case, seed):
    st = State()
    st.case, st.kind = case, case["kind"]
    if st.kind in ("norm", "rows"):
        S, D = case["tokens"], case["width"]
        st.x, st.res, st.w = _rows(case, seed)
        st.sum = torch.empty(S, D, dtype=st.x.dtype, device="cuda")
        st.q = torch.empty(S, _ceil(D) * BLK, dtype=torch.float8_e4m3fn, device="cuda")
        st.s = torch.empty(_ceil(D), S, device="cuda")
    elif st.kind == "product":
        wq, ws, st.xq, st.xs = _product_inputs(case, seed)
        st.y = torch.empty(case["tokens"], case["rows"], dtype=TYPES[case["dtype"]], device="cuda")
        if own:                  # the library lays weights out once, when it is given them
            import zunzuncito_amd as zz
            zz.init()
            st.handle = zz.Fp8Matrix(case["rows"], case["cols"])
            torch.cuda.synchronize()
            st.handle.upload_dev(wq.data_ptr(), ws.data_ptr())
        else:
            st.wq, st.ws = wq, ws
    else:
        N, W = case["seqs"], case["beams"]
        st.logits, st.score, st.done, st.src = _beam_inputs(case, seed)
        st.dst = torch.zeros_like(st.src)
        st.score2 = torch.empty(N, W, device="cuda")
        st.parent = torch.empty(N, W, dtype=torch.int32, device="cuda")
        st.token = torch.empty(N, W, dtype=torch.int32, device="cuda")
        st.done2 = torch.empty(N, W, dtype=torch.bool, device="cuda")
        st.ws = torch.empty(N * W * (case["vocab"] // 8 + 65536), dtype=torch.uint8, device="cuda")
    if own:
        import zunzuncito_amd as zz
        zz.init()
    return st


# ------------------------------------------------------------------ the plain forms
def _plain_rows(y, D):
    b = torch.nn.functional.pad(y, (0, _ceil(D) * BLK - D)).view(y.shape[0], -1, BLK)
    s = b.abs().amax(2).clamp_min(FLOOR) / FMAX
    q = (b / s[:, :, None]).to(torch.float8_e4m3fn).view(y.shape[0], -1)
    return q, s.t().contiguous()


def _plain_norm(st):
    D = st.case["width"]
    x = st.x[:, :D].float()
    if st.kind == "rows":
        q, s = _plain_rows(x, D)
        return dict(q=q, s=s)
    h = x + st.res[:, :D].float()
    q, s = _plain_rows(h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * st.w, D)
    return dict(sum=h.to(st.x.dtype), q=q, s=s)


def _plain_product(st):
    O, I = st.case["rows"], st.case["cols"]
    x = st.xq[:, :I].float() * st.xs.t().repeat_interleave(BLK, 1)[:, :I]
    w = st.wq.float() * st.ws.repeat_interleave(BLK, 0)[:O].repeat_interleave(BLK, 1)[:, :I]
    return dict(y=(x @ w.t()).to(st.y.dtype))


def _plain_beam(st):
    """The sums in 64 bits: neighbouring totals decide the order. A row's candidates go by
    (logit, lower token): their 64-bit keys are all different, so their order is too."""
    c = st.case
    N, W, V = c["seqs"], c["beams"], c["vocab"]
    k = min(W, V)
    L = st.logits.float() + 0.0                              # minus zero counts as zero
    L = torch.where(L.isnan(), -math.inf, L)
    top = L.amax(1, keepdim=True).double()
    lse = top + torch.where(L == top, 1.0, torch.exp(L.double() - top)).sum(1, keepdim=True).log()
    bits = L.view(torch.int32).long()
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    keys = ((order << 32) | (0xFFFFFFFF - torch.arange(V, device="cuda"))).topk(k, dim=1)[0]
    token = 0xFFFFFFFF - (keys & 0xFFFFFFFF)
    total = st.score.double().view(-1, 1) - lse + L.gather(1, token).double()
    total = torch.where(total.isnan(), -math.inf, total).view(N, W, k)
    # a finished beam offers itself alone
    first = torch.arange(k, device="cuda") == 0
    done = st.done[:, :, None]
    total = torch.where(done, torch.where(first, st.score.double()[:, :, None], -math.inf), total)
    live = (~done | first).view(N, W * k)
    token = torch.where(done, 0, token.view(N, W, k)).view(N, W * k)
    # the best W of a sequence: larger total, then the lower beam, then the row's own order
    a = torch.argsort((~live).long(), dim=1, stable=True)    # what is no candidate goes last
    t = total.view(N, W * k).gather(1, a)
    t = torch.where(live.gather(1, a), t, -math.inf)
    b = torch.argsort(t, dim=1, descending=True, stable=True)[:, :W]
    at = a.gather(1, b)
    parent = at // k
    token = token.gather(1, at)
    dst = st.src.view(c["layers"], N, W, c["cap"], c["width"])[:, :, :, :c["len"]]
    dst = dst[:, torch.arange(N, device="cuda")[:, None], parent].reshape(c["layers"], N * W, c["len"], c["width"])
    return dict(score=t.gather(1, b).float(), parent=parent.int(), token=token.int(),
                done=st.done.gather(1, parent) | (token == 1), states=dst)


# ------------------------------------------------------------------ the calls
def _own(st):
    import zunzuncito_amd as zz
    c = st.case
    stream = torch.cuda.current_stream().cuda_stream
    if st.kind == "product":
        st.handle.matmul_dev(st.xq.data_ptr(), st.xs.data_ptr(), c["tokens"], st.y.data_ptr(),
                             dtype=zz.ZZ_F32 if c["dtype"] == "f32" else zz.ZZ_BF16, stream=stream)
        return dict(y=st.y)
    t = zz.ZZ_F32 if c["dtype"] == "f32" else zz.ZZ_BF16
    if st.kind == "rows":
        zz.rows_fp8_dev(st.x.data_ptr(), c["tokens"], c["width"], st.q.data_ptr(), st.s.data_ptr(), dtype=t,
                        ldx=st.x.stride(0), stream=stream)
        return dict(q=st.q, s=st.s)
    if st.kind == "norm":
        zz.add_norm_fp8_dev(st.x.data_ptr(), st.res.data_ptr(), st.sum.data_ptr(), st.w.data_ptr(), c["tokens"],
                            c["width"], EPS, st.q.data_ptr(), st.s.data_ptr(), dtype=t, ldx=st.x.stride(0),
                            ldr=st.res.stride(0), stream=stream)
        return dict(sum=st.sum, q=st.q, s=st.s)
    N, W, esz = c["seqs"], c["beams"], st.src.element_size()
    row = c["cap"] * c["width"] * esz
    zz.beam_step_dev(st.logits.data_ptr(), N, W, c["vocab"], st.score.data_ptr(), st.score2.data_ptr(),
                     st.parent.data_ptr(), st.token.data_ptr(), st.ws.data_ptr(), st.ws.numel(),
                     d_done=st.done.data_ptr(), d_done_out=st.done2.data_ptr(), eos=1, pad=0, dtype=t, stream=stream)
    zz.beam_reorder_dev(st.dst.data_ptr(), st.src.data_ptr(), st.parent.data_ptr(), N, W, outer=c["layers"],
                        outer_stride=N * W * row, row_stride=row, row_bytes=c["len"] * c["width"] * esz, stream=stream)
    return dict(score=st.score2, parent=st.parent, token=st.token, done=st.done2, states=st.dst[:, :, :c["len"]])


def run(st):
    if own:
        return _own(st)
    if st.kind == "product":
        return _plain_product(st)
    return _plain_beam(st) if st.kind == "beam" else _plain_norm(st)


# ------------------------------------------------------------------ work
def work(case):
    esz = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("norm", "rows"):
        S, D = case["tokens"], case["width"]
        streams = 3 if case["kind"] == "norm" else 1
        return {"bytes": S * (D * esz * streams + _ceil(D) * (BLK + 4)) + (4 * D if streams == 3 else 0),
                "flops": 8.0 * S * D}
    if case["kind"] == "product":
        S, O, I = case["tokens"], case["rows"], case["cols"]
        return {"bytes": O * I + 4 * _ceil(O) * _ceil(I) + S * _ceil(I) * (BLK + 4) + S * O * esz,
                "flops": 2.0 * S * O * I}
    R = case["seqs"] * case["beams"]
    k = case["done"] if not case["first"] else 0
    live = R - (R // k if k else 0)              # finished beams' logits need not be read
    moved = 2 * R * case["layers"] * case["len"] * case["width"] * 2
    return {"bytes": live * case["vocab"] * esz + moved + 18 * R, "flops": 4.0 * live * case["vocab"]}


# ------------------------------------------------------------------ 64-bit results
def _e4m3(v):
    """The nearest e4m3 value, ties to even: three bits behind the leading one, steps of
    2^-9 below 2^-6."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _exact_rows(y):
    S, D = y.shape
    q = torch.zeros(S, _ceil(D) * BLK, dtype=torch.float64, device=y.device)
    q[:, :D] = y
    q = q.view(S, _ceil(D), BLK)
    s = torch.maximum(q.max(2)[0], -q.min(2)[0]).clamp_min(FLOOR) / FMAX
    return _e4m3(q / s.unsqueeze(2)).flatten(1), s.t()


def exact(case, seed):
    if case["kind"] in ("norm", "rows"):
        D = case["width"]
        x, res, w = (v.double() for v in _rows(case, seed))
        x, res = x[:, :D], res[:, :D]
        if case["kind"] == "rows":
            q, s = _exact_rows(x)
            return dict(q=q, s=s)
        h = x + res
        q, s = _exact_rows(h / torch.sqrt((h * h).sum(1) / D + EPS)[:, None] * w)
        return dict(sum=h, q=q, s=s)
    if case["kind"] == "product":
        O, I = case["rows"], case["cols"]
        wq, ws, xq, xs = _product_inputs(case, seed)
        y = torch.zeros(case["tokens"], O, dtype=torch.float64, device="cuda")
        for b in range(_ceil(I)):                            # block by block, as it is defined
            at = slice(b * BLK, min(I, (b + 1) * BLK))
            part = xq[:, at].double() @ wq[:, at].double().t()
            y += part * xs[b].double()[:, None] * ws[:, b].double().repeat_interleave(BLK)[None, :O]
        return dict(y=y)
    N, W, V = case["seqs"], case["beams"], case["vocab"]
    logits, score, done, states = _beam_inputs(case, seed)
    score_, states_ = [], []
    for n in range(N):
        total = torch.log_softmax(logits[n * W:(n + 1) * W].double(), 1) + score[n].double()[:, None]
        total[done[n]] = -math.inf
        total[done[n], 0] = score[n][done[n]].double()
        best, at = total.view(-1).topk(W)
        score_.append(best)
        states_.append(states[:, n * W:(n + 1) * W, :case["len"]][:, at // V])
    # beams at minus infinity have no order of their own: the definition's ties decide it
    tied = bool(torch.isinf(torch.stack(score_)).any())
    return dict(score=torch.stack(score_), parent=None, token=None, done=None,
                states=None if tied else torch.cat(states_, 1).double())
