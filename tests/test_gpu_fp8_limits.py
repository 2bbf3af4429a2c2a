"""The fp8 product's far limits: the largest gated pairs, results, rows by index and rows."""
import pytest
import torch

import zunzuncito_amd as zz
from test_gpu_experts import BF16, F32, KIND, ptr, stream
from test_gpu_fp8_sums import Whole

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _up():
    zz.init()


def free(gb):
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0] >= gb << 30


# 2^35 packed codes and more are laid out by more threads than one launch holds
@pytest.mark.parametrize("O, I", [((1 << 19) - 1, 1 << 16), (1 << 24, 2047)])
def test_largest_gated_pair(O, I):
    if not free(130):
        pytest.skip("needs 130 GiB of device memory")
    nb, no = -(-I // 128), -(-O // 128)
    codes = torch.zeros(O, I, dtype=torch.uint8, device="cuda")
    rows = [0, 15, 16, 12345, O // 2, O - 2, O - 1]
    codes[rows] = 0x38                                    # 1.0
    ws = torch.full((no, nb), 1.0 / I, device="cuda")
    mat = zz.Fp8Experts(1, O, I, gated=True)
    try:
        torch.cuda.synchronize()
        mat.upload_dev(0, ptr(codes), ptr(ws))
        codes[rows[3]] = 0
        ws *= 2.0
        torch.cuda.synchronize()
        mat.upload_dev(0, ptr(codes), ptr(ws), part=1)
        del codes
        q = torch.zeros(2, nb * 128, dtype=torch.uint8, device="cuda")
        q[:, :I] = 0x38
        s = torch.tensor([1.0, 4.0], device="cuda").expand(nb, 2).contiguous()
        bias = torch.zeros(2, O, device="cuda")
        bias[1] = 0.5                                     # up's: a column without codes is gate's 0 times a half
        y = torch.full((3, O), 9.0, device="cuda")
        mat.matmul_ep_dev(ptr(q), ptr(s), 2, ptr(y), d_bias=ptr(bias), stream=stream())
        want = torch.zeros(2, O, device="cuda")
        want[0, rows], want[1, rows] = 2.5, 4.0 * 8.5
        want[0, rows[3]], want[1, rows[3]] = 0.5, 2.0
        assert (y[2] == 9.0).all()
        assert (y[:2] - want).abs().max() <= 34.0 * 2 * (I + nb) * 2.0 ** -24
        assert ((y[:2] != 0) == (want != 0)).all()
    finally:
        mat.close()
        torch.cuda.empty_cache()


def test_most_tiles():
    """Results of 2^24 tiles are declined, and why, before anything is launched."""
    mat = zz.Fp8Experts(1, 8191, 5, gated=True)
    try:
        for part in range(2):
            codes, ws = torch.zeros(8191, 5, dtype=torch.uint8, device="cuda"), torch.ones(64, 1, device="cuda")
            torch.cuda.synchronize()
            mat.upload_dev(0, ptr(codes), ptr(ws), part=part)
        far = [1 << 40, 1 << 41, 1 << 42, 1 << 43]        # pretended addresses
        with pytest.raises(RuntimeError, match="2\\^24 tiles"):
            mat.matmul_dev(far[0], far[1], 1 << 24, 0, far[2], 1 << 24, far[3], dtype=zz.ZZ_BF16, stream=stream())
    finally:
        mat.close()


@pytest.mark.parametrize("dtype, S, D", [(torch.bfloat16, (1 << 20) + 77, 130), (torch.float32, (1 << 20) + 1, 1000),
                                         (torch.bfloat16, 1 << 24, 96)])
def test_rows_past_2_20_and_their_product(dtype, S, D):
    """As many rows as a table's product takes: their codes are those of the rows in two calls, and the
    product of them with a table is right at both ends."""
    nb, kind = -(-D // 128), zz.ZZ_BF16 if dtype == torch.bfloat16 else zz.ZZ_F32
    x = torch.randn(S, D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dtype)
    q, s = torch.full((S + 1, nb * 128), 9, dtype=torch.uint8, device="cuda"), torch.full((nb * S + 1,), 9.0, device="cuda")
    zz.rows_fp8_dev(ptr(x), S, D, ptr(q), ptr(s), dtype=kind, stream=stream())
    assert (q[S] == 9).all() and s[nb * S] == 9.0
    cut = list(range(0, S, 1 << 20)) + [S]
    for lo, hi in list(zip(cut, cut[1:])):
        n = hi - lo
        q1, s1 = torch.empty(n, nb * 128, dtype=torch.uint8, device="cuda"), torch.empty(nb, n, device="cuda")
        zz.rows_fp8_dev(x[lo:].data_ptr(), n, D, ptr(q1), ptr(s1), dtype=kind, stream=stream())
        assert torch.equal(q[lo:hi], q1) and torch.equal(s[:nb * S].view(nb, S)[:, lo:hi], s1)
    E, O = 3, 17
    w = torch.randint(0, 100, (E, O, D), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda", dtype=torch.uint8)
    ws = torch.ones(1, nb, device="cuda")
    mat = zz.Fp8Experts(E, O, D)
    try:
        torch.cuda.synchronize()
        for e in range(E):
            mat.upload_dev(e, w[e].data_ptr(), ptr(ws))
        offs = [0, 5, S - 7, S]
        y, cut = torch.empty(S, O, device="cuda"), torch.tensor(offs, dtype=torch.int32).cuda()
        mat.matmul_dev(ptr(q), ptr(s), S, 0, ptr(cut), S, ptr(y), stream=stream())
        f8 = torch.float8_e4m3fn
        for e, at in ((0, slice(0, 5)), (1, slice(5, 40)), (1, slice(S - 40, S - 7)), (2, slice(S - 7, S))):
            rows = q[at].view(f8).double() * s[:nb * S].view(nb, S)[:, at].t().repeat_interleave(128, 1).double()
            v = w[e].view(f8).double()
            off = (y[at].double() - rows[:, :D] @ v.t()).abs()
            assert (off <= (2 * 128 + nb + 18) * 2.0 ** -24 * (rows[:, :D].abs() @ v.t().abs())).all()
    finally:
        mat.close()


@pytest.mark.parametrize("dtype, eight, P, O", [(F32, 0, 9, 33), (BF16, 0, 9, 33), (F32, 0, 300, 200), (BF16, 0, 300, 200), (F32, 0, 4000, 1030),
                                                (BF16, 0, 4000, 1030), (BF16, zz.ZZ_EP_8BIT, 4000, 1030), (BF16, zz.ZZ_EP_8BIT, 9000, 2050)])
def test_rows_by_index_up_to_2_32_bytes(dtype, eight, P, O):
    """Codes of just under 2^32 bytes, of which only the first rows, the last and those on both sides of
    2^31 are named; every other row's are NaN."""
    E, I, n = 2, 1 << 16, (1 << 16) - 1
    c = Whole(E, 1, O, I, n, 3, big=not eight)
    try:
        assert (1 << 32) - (1 << 16) == c.q.numel()
        named = torch.tensor([0, 1, 32766, 32767, 32768, 32769, n - 2, n - 1], device="cuda")
        keep = c.q[named].clone()
        c.q.fill_(0x7F)
        c.q[named] = keep
        at = named[torch.randint(0, 8, (P,), generator=torch.Generator().manual_seed(1)).cuda()]
        at[:8], at[P - 8:] = named, named
        row, offs = at.int(), torch.tensor([0, P // 3, P], dtype=torch.int32).cuda()
        y = torch.full((P + 1, O), 9.0, dtype=dtype, device="cuda")
        c.mat.matmul_dev(ptr(c.q), ptr(c.s), n, ptr(row), ptr(offs), P, ptr(y), act=eight, dtype=KIND[dtype], stream=stream())
        e = (torch.arange(P, device="cuda") >= P // 3).long()
        assert torch.equal(y[:P], c.want(at, e, dtype)) and (y[P] == 9.0).all()
    finally:
        c.mat.close()
