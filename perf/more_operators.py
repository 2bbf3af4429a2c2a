"""Experts of 8-bit floating point, measured against their plain forms: tokens sorted by
expert and back with the routing weights (and the gradients of both), the product with bias,
activation and residual in its epilogue, and the same product over a table of experts.

What a mixture-of-experts layer does with the router's choice: the (token, slot) pairs go
into the experts' order and the tokens' rows with them (kind "dispatch"); each expert's rows
meet its matrix (kind "experts"; "linear" is one matrix for all rows, as of a dense branch);
the results come back, weighted and added up (kind "back"; "grad" is the way back's and the
gathering's gradient together).

Widths, expert counts and choices per token are those of this repository's layers (2816 / 704
with 8 of 128, 2048 / 1792 with 4 of 32, 2048 / 768 with 8 of 256, the dense 2112), and
generic ones.
"""
import math

import torch

own = False

BLK = 128
FMAX = 448.0                     # the largest e4m3 value
FLOOR = 2.0 ** -100              # a block's largest magnitude counts as at least this
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token on its way to 8 experts: a call's latency
        dict(name="dispatch_decode_1", kind="dispatch", tokens=1, top=8, experts=128, width=2816, dtype="f32", drop=0),
        # a serving batch with every fifth choice dropped (an expert at its capacity)
        dict(name="dispatch_batch_37", kind="dispatch", tokens=37, top=4, experts=32, width=2048, dtype="bf16", drop=5),
        # a long prompt over many experts
        dict(name="dispatch_prefill_8192", kind="dispatch", tokens=8192, top=8, experts=256, width=2048, dtype="bf16",
             drop=0),
        # a serving batch's results back onto the residual stream
        dict(name="back_batch_21", kind="back", tokens=21, top=8, experts=128, width=2816, dtype="f32", drop=0, res=True),
        # a long prompt's results
        dict(name="back_prefill_8192", kind="back", tokens=8192, top=8, experts=128, width=2816, dtype="bf16", drop=0,
             res=True),
        # a small training batch, an odd width, dropped choices
        dict(name="grad_batch_50", kind="grad", tokens=50, top=4, experts=32, width=1087, dtype="f32", drop=7),
        # a training batch
        dict(name="grad_train_4096", kind="grad", tokens=4096, top=8, experts=128, width=2816, dtype="bf16", drop=0),
        # one token through a dense down projection, bias and residual with it
        dict(name="linear_decode_1", kind="linear", tokens=1, rows=2816, cols=2112, gated=False, act="none", bias=True,
             res=True, clamp=0.0, dtype="f32"),
        # a prompt through a dense branch's gate and up, their activation with it
        dict(name="linear_prefill_2048", kind="linear", tokens=2048, rows=2112, cols=2816, gated=True, act="gelu",
             bias=False, res=False, clamp=0.0, dtype="bf16"),
        # one token through 8 of 128 experts' gate and up: their matrices' bytes
        dict(name="experts_decode_1", kind="experts", tokens=1, top=8, experts=128, rows=704, cols=2816, gated=True,
             act="gelu", bias=False, res=False, clamp=0.0, dtype="bf16", drop=0, indexed=True),
        # a ragged serving batch through the experts' down matrices, rows in the experts' order
        dict(name="experts_batch_45", kind="experts", tokens=45, top=4, experts=32, rows=2048, cols=1792, gated=False,
             act="none", bias=True, res=False, clamp=0.0, dtype="f32", drop=9, indexed=False),
        # a long prompt through the experts' gate and up, some experts far busier than others
        dict(name="experts_prefill_4096", kind="experts", tokens=4096, top=8, experts=128, rows=704, cols=2816, gated=True,
             act="silu", bias=False, res=False, clamp=7.0, dtype="bf16", drop=0, indexed=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _epilogue(rng):
    gated = rng.random() < 0.5
    return dict(gated=gated, act=rng.choice(["gelu", "silu"] if gated else ["none", "none", "gelu", "silu"]),
                bias=rng.random() < 0.5, res=rng.random() < 0.4,
                clamp=rng.choice([0.0, 7.0]) if gated else 0.0)


def draw(rng):
    kind = rng.choice(["dispatch", "back", "grad", "linear", "linear", "experts", "experts", "experts"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "linear":
        rows, cols = _log_int(rng, 64, 4224), _log_int(rng, 64, 4224)
        tokens = _log_int(rng, 1, min(4096, 2048 * 2 * 2112 * 2816 // (2 * rows * cols)))
        return dict(kind=kind, tokens=tokens, rows=rows, cols=cols, dtype=dtype, **_epilogue(rng))
    experts = _log_int(rng, 1, 512)
    top = rng.randint(1, min(16, experts))
    drop = rng.choice([0, 0, 3, 10])
    if kind == "experts":
        experts = min(experts, 256)
        top = min(top, 8)
        rows = _log_int(rng, 32, 2816)
        cols = _log_int(rng, 64, max(64, min(4096, 128 * 704 * 2816 // (experts * rows))))
        tokens = _log_int(rng, 1, min(4096, 4096 * 8 * 704 * 2816 // (top * rows * cols),
                                      40_000_000 // (top * rows * (4 if dtype == "f32" else 2))))
        return dict(kind=kind, tokens=tokens, top=top, experts=experts, rows=rows, cols=cols, dtype=dtype, drop=drop,
                    indexed=rng.random() < 0.5, **_epilogue(rng))
    width = _log_int(rng, 64, 8192)
    esz = 4 if dtype == "f32" else 2
    tokens = _log_int(rng, 1, min(8192, 590_000_000 // (width * (3 * top + 2) * esz)))
    case = dict(kind=kind, tokens=tokens, top=top, experts=experts, width=width, dtype=dtype, drop=drop)
    return dict(case, res=rng.random() < 0.5) if kind == "back" else case


# ------------------------------------------------------------------ inputs
class State:
    """What a program holds between calls; a table's handle is given back with it."""
    handle = None

    def __del__(self):
        if self.handle is not None:
            self.handle.close()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _routing(case, g):
    """ids [S, K], distinct in a token and skewed over the experts, some dropped (-1); the
    pairs' positions, the tokens at the positions, the experts' offsets."""
    S, K, E = case["tokens"], case["top"], case["experts"]
    skew = -1.1 * torch.log(1.0 + torch.arange(E, device="cuda"))[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand(S, E, generator=g, device="cuda").clamp_min(1e-20)
    ids = (skew - torch.log(-torch.log(u).clamp_min(1e-20))).topk(K, dim=1)[1].int()
    if case["drop"]:
        ids.view(-1)[case["drop"] - 1::case["drop"]] = -1
    w = torch.rand(S, K, generator=g, device="cuda")
    w = w / w.sum(1, keepdim=True)
    return ids, w


def _sorted(ids, E):
    """(offs [E + 1], row [S * K], pos [S, K]) of the ids, what is behind the last pair 0."""
    S, K = ids.shape
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), E, flat)
    at = torch.sort(key, stable=True)[1]
    count = (key[:, None] == torch.arange(E, device=ids.device)).sum(0) if S * K * E <= 1 << 24 else \
        torch.zeros(E + 1, dtype=torch.long, device=ids.device).scatter_add_(0, key, torch.ones_like(key))[:E]
    offs = torch.zeros(E + 1, dtype=torch.int32, device=ids.device)
    offs[1:] = count.cumsum(0)
    place = torch.empty_like(at)
    place[at] = torch.arange(S * K, device=ids.device)
    kept = key < E
    pos = torch.where(kept, place, -1).int().view(S, K)
    row = torch.where(torch.arange(S * K, device=ids.device) < offs[E], at // K, 0).int()
    return offs, row, pos


def _stream_rows(n, D, dtype, g, size=1.0):
    """Rows of a residual stream: some columns far larger than the rest."""
    col = 1 + 9 * (torch.rand(D, generator=g, device="cuda") < 0.01)
    return (size * torch.randn(n, D, generator=g, device="cuda") * col).to(TYPES[dtype])


def _ceil(n):
    return -(-n // BLK)


def _coded(v, br):
    """e4m3 codes of matrices [.., O, I] and the f32 scales of their br x 128 blocks."""
    O, I = v.shape[-2:]
    p = torch.nn.functional.pad(v, (0, _ceil(I) * BLK - I, 0, -(-O // br) * br - O))
    b = p.view(*v.shape[:-2], p.shape[-2] // br, br, _ceil(I), BLK)
    s = b.abs().amax((-3, -1)).clamp_min(FLOOR) / FMAX
    q = (b / s[..., :, None, :, None]).view(p.shape).to(torch.float8_e4m3fn)
    return q[..., :O, :], s


def _table(case, g):
    """Codes [E, parts, O, I] (gate and up of a gated table), scales and bias."""
    E, O, I, G = case.get("experts", 1), case["rows"], case["cols"], 2 if case["gated"] else 1
    wq = torch.empty(E, G, O, I, dtype=torch.float8_e4m3fn, device="cuda")
    ws = torch.empty(E, G, _ceil(O), _ceil(I), device="cuda")
    step = max(1, (1 << 27) // (G * O * I))
    for e in range(0, E, step):
        n = min(step, E - e)
        q, ws[e:e + n] = _coded(torch.empty(n, G, O, I, device="cuda").normal_(0.0, 1.0 / math.sqrt(I), generator=g), BLK)
        wq[e:e + n] = q[..., :I]
    bias = 0.3 * torch.randn(E, G, O, generator=g, device="cuda") if case["bias"] else None
    return wq, ws, bias


def _product_inputs(case, seed):
    g = _gen(seed)
    st = State()
    st.wq, st.ws, st.bias = _table(case, g)
    S, P = case["tokens"], case["tokens"]
    st.offs = st.row = None
    if case["kind"] == "experts":
        ids, _ = _routing(case, g)
        P = ids.numel()
        st.offs, st.row, _ = _sorted(ids, case["experts"])
        if not case["indexed"]:
            S, st.row = P, None
    col = 1 + 9 * (torch.rand(case["cols"], generator=g, device="cuda") < 0.01)
    q, s = _coded(torch.randn(S, case["cols"], generator=g, device="cuda") * col, 1)
    st.xq, st.xs = q.contiguous(), s.t().contiguous()
    st.res = _stream_rows(P, case["rows"], case["dtype"], g, 2.0) if case["res"] else None
    st.P = P
    return st


def _way_inputs(case, seed):
    """The routing, and rows in the tokens' and in the experts' order."""
    g = _gen(seed)
    st = State()
    S, K, D, t = case["tokens"], case["top"], case["width"], case["dtype"]
    st.ids, st.w = _routing(case, g)
    st.x = _stream_rows(S, D, t, g, 2.0)
    if case["kind"] == "dispatch":
        return st
    _, _, st.pos = _sorted(st.ids, case["experts"])
    st.y = _stream_rows(S * K, D, t, g)
    if case["kind"] == "grad":
        st.dxs = _stream_rows(S * K, D, t, g)
    return st


def prepare(case, seed):
    if case["kind"] in ("linear", "experts"):
        st = _product_inputs(case, seed)
        # what lies behind the last expert's rows stays as it is
        st.y = torch.zeros(st.P, case["rows"], dtype=TYPES[case["dtype"]], device="cuda")
        if own:                  # the library lays the codes out once, when it is given them
            import zunzuncito_amd as zz
            zz.init()
            E, G = st.wq.shape[:2]
            st.handle = zz.Fp8Experts(E, case["rows"], case["cols"], gated=case["gated"])
            torch.cuda.synchronize()
            for e in range(E):
                for part in range(G):
                    st.handle.upload_dev(e, st.wq[e, part].data_ptr(), st.ws[e, part].data_ptr(), part=part)
            st.wq = st.ws = None
    else:
        st = _way_inputs(case, seed)
        S, K, D, t = case["tokens"], case["top"], case["width"], TYPES[case["dtype"]]
        if case["kind"] == "dispatch":
            st.offs = torch.empty(case["experts"] + 1, dtype=torch.int32, device="cuda")
            st.row = torch.zeros(S * K, dtype=torch.int32, device="cuda")
            st.pos = torch.empty(S, K, dtype=torch.int32, device="cuda")
            st.xs = torch.zeros(S * K, D, dtype=t, device="cuda")
            if own:
                import zunzuncito_amd as zz
                zz.init()
                st.ws = torch.empty(zz.experts_ws_bytes(S, K, case["experts"]), dtype=torch.uint8, device="cuda")
        else:
            st.out = torch.empty(S, D, dtype=t, device="cuda")
            st.dy = torch.zeros(S * K, D, dtype=t, device="cuda")
            st.dw = torch.empty(S, K, device="cuda")
    st.case = case
    if own:
        import zunzuncito_amd as zz
        zz.init()
    return st


# ------------------------------------------------------------------ the plain forms
def _take(rows, pos):
    """The rows [S, K, D] at the positions in 32 bits, zeros for what was dropped."""
    kept = pos >= 0
    v = rows.float()[torch.where(kept, pos, 0).long()]
    return torch.where(kept[:, :, None], v, 0.0)


def _put(pos, v, dtype):
    """v [S, K, D] at its positions, zeros behind the last one."""
    S, K, D = v.shape
    out = torch.zeros(S * K + 1, D, dtype=dtype, device=v.device)
    out[torch.where(pos >= 0, pos, S * K).long().view(-1)] = v.reshape(S * K, D).to(dtype)
    return out[:S * K]


def _plain_way(st):
    c = st.case
    S, K, D = c["tokens"], c["top"], c["width"]
    if c["kind"] == "dispatch":
        offs, row, pos = _sorted(st.ids, c["experts"])
        return dict(offs=offs, row=row, pos=pos, xs=_put(pos, st.x[:, None].expand(S, K, D), st.x.dtype))
    if c["kind"] == "back":
        out = (_take(st.y, st.pos) * st.w[:, :, None]).sum(1)
        return dict(out=(out + st.x.float() if c["res"] else out).to(st.y.dtype))
    dout = st.x.float()[:, None]
    return dict(dy=_put(st.pos, dout * st.w[:, :, None], st.y.dtype), dw=(_take(st.y, st.pos) * dout).sum(2),
                dx=_take(st.dxs, st.pos).sum(1).to(st.y.dtype))


def _activated(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v / (1.0 + torch.exp(-v)) if act == "silu" else v


def _ended(parts, c):
    """The activation of one matrix' sums, or of gate's and up's."""
    if not c["gated"]:
        return _activated(parts[0], c["act"])
    gate, up = parts
    if c["clamp"] > 0:
        gate, up = gate.clamp_max(c["clamp"]), up.clamp(-c["clamp"], c["clamp"])
    return _activated(gate, c["act"]) * up


def _plain_product(st):
    c = st.case
    E, G, O, I = st.wq.shape
    x = st.xq[:, :I].float() * st.xs.t().repeat_interleave(BLK, 1)[:, :I]
    offs = [0, st.P] if st.offs is None else st.offs.tolist()
    y = torch.zeros(st.P, O, dtype=st.y.dtype, device=x.device)
    for e in range(E):
        at = slice(offs[e], offs[e + 1])
        if at.start == at.stop:
            continue
        rows = x[at] if st.row is None else x[st.row[at].long()]
        w = st.wq[e].float() * st.ws[e].repeat_interleave(BLK, 1)[:, :O].repeat_interleave(BLK, 2)[:, :, :I]
        v = _ended([rows @ w[i].t() + (0.0 if st.bias is None else st.bias[e, i]) for i in range(G)], c)
        y[at] = (v if st.res is None else v + st.res[at].float()).to(y.dtype)
    return dict(y=y)


# ------------------------------------------------------------------ the calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own(st):
    import zunzuncito_amd as zz
    c = st.case
    t = zz.ZZ_F32 if c["dtype"] == "f32" else zz.ZZ_BF16
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] in ("linear", "experts"):
        ep = dict(d_bias=_ptr(st.bias), act={"none": zz.ZZ_EP_NONE, "gelu": zz.ZZ_EP_GELU_TANH, "silu": zz.ZZ_EP_SILU}[c["act"]],
                  clamp=c["clamp"], d_res=_ptr(st.res), dtype=t, stream=stream)
        if c["kind"] == "linear":
            st.handle.matmul_ep_dev(st.xq.data_ptr(), st.xs.data_ptr(), st.P, st.y.data_ptr(), **ep)
        else:
            st.handle.matmul_dev(st.xq.data_ptr(), st.xs.data_ptr(), st.xq.shape[0], _ptr(st.row), st.offs.data_ptr(),
                                 st.P, st.y.data_ptr(), **ep)
        return dict(y=st.y)
    S, K, D = c["tokens"], c["top"], c["width"]
    if c["kind"] == "dispatch":
        zz.experts_dispatch_dev(st.ids.data_ptr(), S, K, c["experts"], st.offs.data_ptr(), st.row.data_ptr(),
                                st.pos.data_ptr(), st.ws.data_ptr(), st.ws.numel(), d_x=st.x.data_ptr(), D=D,
                                d_xs=st.xs.data_ptr(), dtype=t, stream=stream)
        return dict(offs=st.offs, row=st.row, pos=st.pos, xs=st.xs)
    if c["kind"] == "back":
        zz.experts_back_dev(st.y.data_ptr(), st.pos.data_ptr(), st.w.data_ptr(), S, K, D, st.out.data_ptr(),
                            d_res=st.x.data_ptr() if c["res"] else 0, dtype=t, stream=stream)
        return dict(out=st.out)
    zz.experts_back_grad_dev(st.x.data_ptr(), st.y.data_ptr(), st.pos.data_ptr(), st.w.data_ptr(), S, K, D,
                             st.dy.data_ptr(), st.dw.data_ptr(), dtype=t, stream=stream)
    # the gathering's gradient is a way back without weights
    zz.experts_back_dev(st.dxs.data_ptr(), st.pos.data_ptr(), 0, S, K, D, st.out.data_ptr(), dtype=t, stream=stream)
    return dict(dy=st.dy, dw=st.dw, dx=st.out)


def run(st):
    if own:
        return _own(st)
    return _plain_product(st) if st.case["kind"] in ("linear", "experts") else _plain_way(st)


# ------------------------------------------------------------------ work
def work(case):
    esz = 4 if case["dtype"] == "f32" else 2
    S, K = case["tokens"], case.get("top", 1)
    P = S * K - (S * K // case["drop"] if case.get("drop") else 0)
    if case["kind"] in ("linear", "experts"):
        O, I, G = case["rows"], case["cols"], 2 if case["gated"] else 1
        E = case.get("experts", 1)
        rows = P if case["kind"] == "experts" and not case["indexed"] else S
        # experts that a uniform choice leaves without rows are not read (a skewed one leaves more)
        used = E if case["kind"] == "linear" else E * (1 - (1 - 1 / E) ** P)
        return {"bytes": used * G * (O * I + 4 * _ceil(O) * _ceil(I)) + rows * _ceil(I) * (BLK + 4) +
                P * O * esz * (2 if case["res"] else 1), "flops": 2.0 * P * G * O * I}
    D = case["width"]
    if case["kind"] == "dispatch":
        return {"bytes": (S + P) * D * esz + 12 * S * K + 4 * case["experts"], "flops": float(S * K)}
    if case["kind"] == "back":
        return {"bytes": (P + S * (2 if case["res"] else 1)) * D * esz + 8 * S * K, "flops": 2.0 * P * D}
    return {"bytes": (3 * P + 2 * S) * D * esz + 12 * S * K, "flops": 4.0 * P * D}


# ------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    if case["kind"] in ("linear", "experts"):
        st = _product_inputs(case, seed)
        E, G, O, I = st.wq.shape
        bounds = [0, st.P] if st.offs is None else st.offs.cpu().tolist()
        y = torch.zeros(st.P, O, dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if lo == hi:
                continue
            rows = torch.arange(lo, hi, device="cuda") if st.row is None else st.row[lo:hi].long()
            sums = []
            for i in range(G):
                total = torch.zeros(hi - lo, O, dtype=torch.float64, device="cuda")
                for b in range(_ceil(I)):                        # block by block, as it is defined
                    cols = slice(b * BLK, min(I, (b + 1) * BLK))
                    part = st.xq[:, cols][rows].double() @ st.wq[e, i, :, cols].double().t()
                    total += part * st.xs[b][rows].double()[:, None] * st.ws[e, i, :, b].double().repeat_interleave(BLK)[None, :O]
                sums.append(total if st.bias is None else total + st.bias[e, i].double())
            gate = sums[0]
            if case["clamp"] > 0:
                gate = torch.minimum(gate, torch.full_like(gate, case["clamp"]))
            if case["act"] == "gelu":                            # half of 1 + tanh is a logistic function
                gate = gate * torch.special.expit(math.sqrt(8.0 / math.pi) * (gate + 0.044715 * gate ** 3))
            elif case["act"] == "silu":
                gate = gate * torch.special.expit(gate)
            if G == 2:
                up = sums[1]
                if case["clamp"] > 0:
                    up = torch.where(up.abs() > case["clamp"], up.sign() * case["clamp"], up)
                gate = gate * up
            y[lo:hi] = gate if st.res is None else gate + st.res[lo:hi].double()
        return dict(y=y)
    st = _way_inputs(case, seed)
    S, K, D = case["tokens"], case["top"], case["width"]
    if case["kind"] == "dispatch":
        key = torch.where(st.ids.view(-1) < 0, case["experts"], st.ids.view(-1)).long()
        order = torch.argsort(key * (S * K) + torch.arange(S * K, device="cuda"))
        xs = st.x[order // K].double()
        xs[int((key < case["experts"]).sum()):] = 0.0
        return dict(offs=None, row=None, pos=None, xs=xs)
    if case["kind"] == "back":
        out = st.x.double() if case["res"] else torch.zeros(S, D, dtype=torch.float64, device="cuda")
        for j in range(K):
            at = st.pos[:, j].long()
            out += torch.where(at >= 0, st.w[:, j].double(), 0.0)[:, None] * st.y[at.clamp_min(0)].double()
        return dict(out=out)
    dy = torch.zeros(S * K, D, dtype=torch.float64, device="cuda")
    dw = torch.zeros(S, K, dtype=torch.float64, device="cuda")
    dx = torch.zeros(S, D, dtype=torch.float64, device="cuda")
    for j in range(K):
        kept = torch.nonzero(st.pos[:, j] >= 0)[:, 0]
        at = st.pos[kept, j].long()
        dout = st.x[kept].double()
        dy[at] = dout * st.w[kept, j].double()[:, None]
        dw[kept, j] = torch.linalg.vecdot(dout, st.y[at].double())
        dx[kept] += st.dxs[at].double()
    return dict(dy=dy, dw=dw, dx=dx)
