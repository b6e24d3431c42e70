"""libsealfm.so holds no kernel of the 4-bit products that no call launches: 32 rows of x a wave are a variant for bf16 (``w4_linear`` of w4_kernels.hip)."""
from seal_amd import _build


def test_kernels_that_no_call_reaches_are_not_built():
    with open(_build.LIB, "rb") as f:
        lib = f.read()
    assert lib.count(b"k_w4_linear_manyI14__hip_bfloat16Li2ELi2E") and lib.count(b"k_w4_linear_manyIfLi2ELi1E")
    assert not lib.count(b"k_w4_linear_manyIfLi2ELi2E")
