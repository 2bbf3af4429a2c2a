"""What a product with an epilogue takes as its activation: one of the three, with or without the
8-bit instructions. Looked at before anything else, so these run without a device."""
import pytest

import zunzuncito_amd as zz

A = 1 << 26                      # pretended device addresses, far apart
Q, S, Y, OFFS = A, 2 * A, 3 * A, 4 * A


def calls(act):
    L = zz.lib()
    yield L.zz_fp8_matmul_ep_dev(-1, Q, S, 4, None, act, 0.0, None, 0, 1, Y, 0, None)
    yield L.zz_fp8_matmul_experts_dev(-1, Q, S, 4, None, OFFS, 4, None, act, 0.0, None, 0, 1, Y, 0, None)


@pytest.mark.parametrize("act", [3, 4, 15, zz.ZZ_EP_8BIT + 3, 2 * zz.ZZ_EP_8BIT, -1, -zz.ZZ_EP_8BIT, 2 ** 31 - 1, -2 ** 31])
def test_other_activations_decline(act):
    for ok in calls(act):
        assert ok == 0 and f"activation {act} declined" in zz.last_error()


@pytest.mark.parametrize("act", [zz.ZZ_EP_NONE, zz.ZZ_EP_GELU_TANH, zz.ZZ_EP_SILU])
def test_activations_pass(act):
    for a in (act, act | zz.ZZ_EP_8BIT):
        for ok in calls(a):       # declined for what comes after: no library, or no such matrix
            assert ok == 0 and any(w in zz.last_error() for w in ("gpu_init", "no such"))


@pytest.mark.parametrize("bad, why", [
    (dict(S=(1 << 24) + 1), "bad arguments"), (dict(S=1 << 24, D=128 * 9), "2\\^27"), (dict(S=1 << 24, ldx=(1 << 36) + 1), "closer"),
    (dict(S=4, ldx=(1 << 40) + 1), "closer"), (dict(S=1 << 24), "overlaps"), (dict(S=1 << 24, ldx=1 << 36), "overlaps"),
])
def test_rows_of_a_table(bad, why):
    """As many rows are rounded as a table's product takes; what is too many, too far apart or overlaps
    (here: the codes and x's rows) is declined."""
    with pytest.raises(RuntimeError, match=why):
        zz.rows_fp8_dev(**{**dict(d_x=Q, S=4, D=1024, d_q=Q + (1 << 30), d_s=1 << 50), **bad})
