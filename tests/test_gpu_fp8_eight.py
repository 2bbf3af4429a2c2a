"""The products with an epilogue where the caller takes the 8-bit matrix instructions (ZZ_EP_8BIT): the
tests of test_gpu_experts.py once more, their calls for bf16 results with it."""
import types

import pytest

import test_gpu_experts as T
import zunzuncito_amd as zz

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _up():
    zz.init()


@pytest.fixture(autouse=True)
def eight(monkeypatch):
    for name in ("matmul_ep_dev", "matmul_dev"):
        def call(self, *args, _plain=getattr(zz.Fp8Experts, name), act=0, dtype=zz.ZZ_F32, **kw):
            return _plain(self, *args, act=act | (zz.ZZ_EP_8BIT if dtype == zz.ZZ_BF16 else 0), dtype=dtype, **kw)
        monkeypatch.setattr(zz.Fp8Experts, name, call)


def again(f):
    """The same test, under its own name here."""
    g = types.FunctionType(f.__code__, f.__globals__, f.__name__, f.__defaults__, f.__closure__)
    g.pytestmark, g.__module__ = list(getattr(f, "pytestmark", [])), __name__
    return g


for _name in ("test_epilogue", "test_epilogue_in_every_form", "test_epilogue_in_tiles_of_any_depth", "test_experts_in_every_form",
              "test_epilogue_large_result", "test_epilogue_strides_and_in_place", "test_epilogue_edges_in_tiles", "test_experts",
              "test_experts_in_the_smaller_forms", "test_experts_far_rows", "test_experts_far_codes", "test_experts_most_rows",
              "test_layer", "test_streams_and_graphs"):
    globals()[_name] = again(getattr(T, _name))


# tables on the 8-bit 64 x 64 tiles too, which only many narrow experts take
@pytest.mark.parametrize("gated, E, P, O, I", [(False, 130, 15554, 33, 3290), (True, 132, 14468, 17, 2353), (False, 17, 1145, 3035, 319),
                                               (True, 4, 257, 6359, 279)])
def test_tables_on_the_8bit_tiles(gated, E, P, O, I):
    T.test_experts_in_every_form(T.BF16, gated, E, P, O, I)
