"""Refusals of the mixture-of-experts entry points that need no GPU: each call fails before it touches the device."""
import ctypes as C

import pytest

from pytorch_b200 import _cabi as cabi


@pytest.fixture(scope="module")
def lib():
    return cabi.lib()


@pytest.mark.parametrize("begin", [-1, -8, -2 ** 63])
def test_a_negative_first_expert(lib, begin):
    """A negative index is a padded token's and has no row: no range takes it in."""
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256
    a = cabi.MoeRouteArgs()
    a.x, a.x_dtype, a.expert_idx, a.idx_dtype, a.tokens, a.topk, a.hidden = p, cabi.BF16, p, cabi.I32, 4, 2, 8
    a.expert_begin, a.expert_end, a.out, a.out_rows, a.row_idx = begin, begin + 8, p, 9, p      # out_rows is wrong too, but checked later
    assert lib.b200q_moe_route(C.byref(a), None) == cabi.ERR_BAD_ARG
    assert "negative expert_begin" in lib.b200q_last_error().decode()
