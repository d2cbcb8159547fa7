"""The launch rule of the 8-bit product, which is the host's: the sizes that the GPU tests give each kernel are its own, and every
kernel is given some in every output type."""
import itertools

import pytest

from tfrec_amd import _lib


def test_the_cases_of_every_kernel_are_its_own():
    pytest.importorskip("torch")
    from test_gpu_int8_kernels import CASES, DT, kernel
    for (which, M, N, K), out in itertools.product(CASES, DT):
        assert kernel(M, N, K, out) == which, (which, M, N, K, out)
    assert {c[0] for c in CASES} == {_lib.I8_ROWS, _lib.I8_SHORT, _lib.I8_TILES_256, _lib.I8_TILES_128, _lib.I8_TILES_128_DEEP}


def test_tiles_need_rows_within_32_bit_offsets():
    lib = _lib.load()
    for M, N, K in ((128, 8193, 1281), (256, 20499, 640), (33, 70001, 520), (4096, 8192, 8192)):
        tiles = (_lib.I8_TILES_256, _lib.I8_TILES_128, _lib.I8_TILES_128_DEEP)
        near, far = (1 << 24) - 16, 1 << 24
        assert lib.tfrec_matmul_i8_kernel(M, N, K, near, near, 0) in tiles
        for lda, ldb in ((far, near), (near, far), (far, far)):
            assert lib.tfrec_matmul_i8_kernel(M, N, K, lda, ldb, 0) not in tiles
