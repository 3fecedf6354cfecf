"""Sizes that the token-step entry points cannot count are refused before any CUDA call (no GPU needed)."""
import ctypes

import pytest

import tadma_b200 as tb
from tadma_b200.abi import DType, Status, make_tensor

FAKE = 0x10000  # never dereferenced: every call fails validation first


def T(dtype, dims, at=FAKE):
    return make_tensor(at, dtype, dims)


@pytest.mark.parametrize("k", [2 ** 31 - 2 ** 14 + 32, 2 ** 31 - 4096, 2 ** 31 - 32, 2 ** 33])
def test_matvec_of_rows_past_the_counters(k):
    args = [T(DType.F16, [1, k]), T(DType.U8, [3, k // 2]), T(DType.F16, [3, k // 32]), tb.none_tensor(), tb.none_tensor(), T(DType.F16, [1, 3])]
    assert tb.lib().tadma_b200_matvec_q4(*map(ctypes.byref, args), None) == Status.ERR_UNSUPPORTED
    assert b"too large" in tb.lib().tadma_b200_last_error()
