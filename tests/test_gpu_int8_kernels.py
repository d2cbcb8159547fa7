"""Every kernel of the 8-bit product, in every output type, at sizes that the launch rule sends to it (asserted, so that a changed
rule cannot empty these tests): ragged tiles, short pipelines, extreme sums, rows far apart, outputs inside a wider matrix."""
import numpy as np
import pytest

from test_gpu_int8 import T, check_product, product_case, quant_rows
from tfrec_amd import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": _lib.DT_F32, "bf16": _lib.DT_BF16, "f16": _lib.DT_F16}

# (kernel, M, N, K), the same for every output type.  The pipeline of four buffers: two steps of 128 columns, three, three whose last
# is cut, and long ones
CASES = [(_lib.I8_TILES_128_DEEP, M, N, K) for M, N, K in ((128, 20000, 256), (128, 20001, 384), (100, 24001, 300), (128, 8193, 1281), (20, 30001, 1030), (300, 5003, 777))] + \
        [(_lib.I8_TILES_128, M, N, K) for M, N, K in ((33, 70001, 520), (130, 40001, 600), (17, 40003, 3000))] + \
        [(_lib.I8_TILES_256, M, N, K) for M, N, K in ((2100, 4701, 600), (129, 41001, 640), (257, 20499, 1041))] + \
        [(_lib.I8_SHORT, M, N, K) for M, N, K in ((1000, 3301, 200), (129, 12701, 20), (70, 30001, 64), (66, 30001, 241))] + \
        [(_lib.I8_ROWS, M, 333, K) for M in (9, 30, 50, 100) for K in (200, 1500, 5000)]
NAMES = {_lib.I8_ROWS: "rows", _lib.I8_SHORT: "short", _lib.I8_TILES_256: "tiles256", _lib.I8_TILES_128: "tiles128", _lib.I8_TILES_128_DEEP: "deep"}


def kernel(M, N, K, out, lda=None, ldb=None):
    pitch = (K + 15) // 16 * 16
    return _lib.load().tfrec_matmul_i8_kernel(M, N, K, lda or pitch, ldb or pitch, DT[out])


def ids(c):
    return "%s-%dx%dx%d" % ((NAMES[c[0]],) + c[1:])


@pytest.fixture(scope="module")
def dev():
    from tfrec_amd.sharded import make_device
    before = torch.cuda.current_stream()
    d = make_device(0)
    yield d
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    d.close()


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=ids)
def test_kernel(dev, case, out):
    which, M, N, K = case
    assert kernel(M, N, K, out) == which
    A, sa, B, sb, b = product_case(M + N + K, M, N, K, bias=K % 2 == 0, full=K % 3 == 0)
    check_product(dev, A, sa * np.float32(0.002), B, sb, b, out)


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [c for c in CASES if c[1:] in ((100, 24001, 300), (33, 70001, 520), (257, 20499, 1041), (66, 30001, 241), (30, 333, 1500), (100, 333, 5000))], ids=ids)
def test_kernel_into_a_pitched_slice(dev, case, out):
    """C's rows start off their 16 bytes and end inside a wider matrix; what lies around them stays."""
    which, M, N, K = case
    assert kernel(M, N, K, out) == which
    A, sa, B, sb, b = product_case(M * 3 + K, M, N, K)
    a, w, bias = quant_rows(A, sa * np.float32(0.002), K), quant_rows(B, sb, K), torch.from_numpy(b).cuda()
    whole = torch.full((M + 2, N + 5), 7.0, dtype=T[out], device="cuda")
    dev.matmul_i8(a, w, bias=bias, out=whole[1:-1, 3:-2])
    want = dev.matmul_i8(a, w, bias=bias, out=torch.empty(M, N, dtype=T[out], device="cuda"))
    dev.synchronize()
    assert torch.equal(whole[1:-1, 3:-2], want)
    whole[1:-1, 3:-2] = 7.0
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("which,M,N,K", [(_lib.I8_TILES_128_DEEP, 130, 3901, 131071), (_lib.I8_TILES_256, 2560, 4099, 131071), (_lib.I8_TILES_128, 128, 33000, 66001),
                                         (_lib.I8_SHORT, 1000, 33001, 511), (_lib.I8_ROWS, 100, 333, 131071)], ids=lambda v: str(v))
def test_extreme_sums_of_every_kernel(dev, which, M, N, K):
    """Rows of -128, 127, -127 and 0 alone: the sums reach 2^31 - 2^14 either way and are exact."""
    from tfrec_amd.device import QuantRows
    assert kernel(M, N, K, "f32") == which
    ld = (K + 15) // 16 * 16
    values = torch.tensor([-128, 127, -127, 0, -128], dtype=torch.int8, device="cuda")
    va, vb = values[torch.arange(M, device="cuda") % 5], values[torch.arange(N, device="cuda") % 5]
    a = QuantRows(va[:, None].expand(M, ld).contiguous(), torch.ones(M, device="cuda"), K)
    b = QuantRows(vb[:, None].expand(N, ld).contiguous(), torch.ones(N, device="cuda"), K)
    C = dev.matmul_i8(a, b, out=torch.empty(M, N, device="cuda"))
    dev.synchronize()
    assert torch.equal(C, (va.double()[:, None] * vb.double()[None, :] * K).float())


@pytest.mark.parametrize("which,ld,M,N,K", [(_lib.I8_TILES_128_DEEP, (1 << 24) - 16, 128, 8193, 1281), (_lib.I8_ROWS, 1 << 24, 128, 8193, 1281),
                                            (_lib.I8_TILES_256, (1 << 24) - 16, 256, 41001, 640), (_lib.I8_SHORT, 1 << 24, 256, 41001, 640)], ids=lambda v: str(v))
def test_rows_just_within_and_just_beyond_32_bit_offsets(dev, which, ld, M, N, K):
    """Row pitches on either side of 16 MiB: up to there a tile's rows are reached by 32-bit offsets (the largest just below
    2^31 or 2^32), beyond other kernels have to take over."""
    from tfrec_amd.device import QuantRows
    assert kernel(M, N, K, "f32", lda=ld) == which and kernel(M, N, K, "f32") in (_lib.I8_TILES_128_DEEP, _lib.I8_TILES_256)
    A, sa, B, sb, b = product_case(7, M, N, K)
    wide = torch.zeros(M, ld, dtype=torch.int8, device="cuda")
    wide[:, :K] = torch.from_numpy(A).cuda()
    a, w, bias = QuantRows(wide, torch.from_numpy(sa).cuda(), K), quant_rows(B, sb, K), torch.from_numpy(b).cuda()
    got, want = (dev.matmul_i8(x, w, bias=bias, out=torch.empty(M, N, device="cuda")) for x in (a, quant_rows(A, sa, K)))
    dev.synchronize()
    assert torch.equal(got, want)
    check_product(dev, A, sa, B, sb, b)
