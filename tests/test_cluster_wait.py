"""A cluster whose CTAs add one another's partial sums stores nothing once a bounded wait of one of them
ran out: the diagnostic runs the W4A4 GEMM's exchange with a CTA that waits (about 1 ms) for an arrival
that never comes."""
import ctypes

import pytest


def test_bad_arguments_are_refused():
    from bitdance_b200 import _lib, build
    build.build_library()
    f = _lib.load().bd_selftest_cluster_wait
    ok = ctypes.c_void_p(4096)  # never dereferenced
    for args in ((10, 2, 0, ok), (1 << 40, 2, 0, ok), (1 << 20, 3, 0, ok), (1 << 20, 16, 0, ok),
                 (1 << 20, 4, 4, ok), (1 << 20, 4, -2, ok), (1 << 20, 4, 0, None)):
        assert f(*args, None) == _lib.BD_ERR_INVALID_ARG
    assert f(1 << 20, 4, 0, ctypes.c_void_p(4098), None) == _lib.BD_ERR_ALIGNMENT


@pytest.mark.gpu
@pytest.mark.parametrize("ctas", [2, 4, 8])
def test_no_cta_stores_beside_one_that_gave_up(ctas):
    import bitdance_b200 as bd
    from bitdance_b200 import _lib, ops
    assert ops.selftest_cluster_wait(ctas) == (0, [1] * ctas)
    for failing in range(ctas):
        word, stored = ops.selftest_cluster_wait(ctas, failing)
        assert word and not word & ~_lib.BD_DEVERR_WAIT_MASK
        assert stored == [0] * ctas
    assert bd.device_error() == 0
