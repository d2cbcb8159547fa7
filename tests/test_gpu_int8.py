"""8-bit rows on the GPU: quantisation, the 8-bit product and the 8-bit top-k, against their definitions in 64 bits (and, where
the order of equal scores matters, in the float32 steps that define a score)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from tfrec_amd.sharded import make_device
    before = torch.cuda.current_stream()
    d = make_device(0)                       # the library's stream is torch's current stream
    yield d
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    d.close()


T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step, relative


def quant_rows(q, s, d):
    """QuantRows on the GPU from host whole numbers [n, d] and scales, padding filled with rubbish."""
    from tfrec_amd.device import QuantRows
    n, ld = q.shape[0], (d + 15) // 16 * 16
    full = np.full((n, ld), 77, np.int8)
    full[:, :d] = q
    return QuantRows(torch.from_numpy(full).cuda(), torch.from_numpy(np.asarray(s, np.float32)).cuda(), d)


# ------------------------------------------------------------------------------------------------------- quantisation
def defined_rows(x64):
    """(q, scale) of rows in double: scale = float32(max|x| / 127), q = nearest-even(x / scale)."""
    top = np.abs(x64).max(1) if x64.shape[1] else np.zeros(len(x64))
    s = (top / 127.0).astype(np.float32)
    with np.errstate(all="ignore"):
        q = np.where(s[:, None] > 0, np.rint(x64 / s.astype(np.float64)[:, None]), 0.0)
    return np.clip(np.nan_to_num(q), -127, 127).astype(np.int8), s


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 15), (5, 16), (7, 17), (65, 20), (33, 64), (4, 100), (9, 257), (3, 1000), (2, 1025), (1, 8192), (3, 20001)])
def test_quantize_matches_the_definition(dev, dtype, n, d):
    g = torch.Generator().manual_seed(n * 1000 + d)
    x = (torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 2)).to(T[dtype])
    if n > 2:
        x[1] = 0.0
    qr = dev.quantize_rows(x.cuda())
    want_q, want_s = defined_rows(x.double().numpy())
    got = qr.q.numpy()
    assert np.array_equal(qr.scale.numpy(), want_s)
    assert np.array_equal(got[:, :d], want_q)
    assert not got[:, d:].any()


def test_quantize_borders_ties_and_extremes(dev):
    """Values on and next to the middle between two whole numbers, subnormal rows, the largest floats, infinities and NaN."""
    s = np.float32(0.37)
    mids = (np.arange(-126, 126) + 0.5).astype(np.float64) * np.float64(s)
    near = mids.astype(np.float32)
    rows = [near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf))]
    x = np.zeros((16, 256), np.float32)
    for i, r in enumerate(rows):
        x[i, :252] = r
        x[i, 255] = np.float32(127) * s
    x[3, :] = np.arange(256) - 128.0          # scale 128 / 127
    x[4, :] = (np.arange(256) - 127.0) / 2    # exact halves of a scale of 64.5 / 127
    x[5, :4] = [127.0, 0.5, 1.5, -2.5]        # scale 1: exact ties to even
    x[6, :3] = [1e-45, -3e-45, 1.4e-43]       # subnormal
    x[7, :3] = [1e-45, 0, 0]                  # scale rounds to zero
    x[8, :3] = [3.4e38, -3.4e38, 1e30]
    x[9, :3] = [1e-38, 2e-38, -3e-39]
    x[10, 3] = np.inf
    x[11, 3] = np.nan
    x[12, :2] = [-np.inf, np.nan]
    x[13, :3] = [2.0 ** -61, 2.0 ** -62, 0.3 * 2.0 ** -61]
    qr = dev.quantize_rows(torch.from_numpy(x).cuda())
    q, sc = qr.q.numpy(), qr.scale.numpy()
    ok = np.r_[0:10, 13:16]
    want_q, want_s = defined_rows(x[ok].astype(np.float64))
    assert np.array_equal(sc[ok], want_s)
    assert np.array_equal(q[ok], want_q)
    assert np.isnan(sc[10:13]).all() and not q[10:13].any()
    assert list(q[5, :4]) == [127, 0, 2, -2]


def test_quantize_listed_rows_pitch_and_bad_ids(dev):
    from tfrec_amd.device import QuantRows
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(40, 90, generator=g).cuda()
    x = wide[:, 3:73]                                        # a pitch, and a base that is only 4-byte aligned
    rows = torch.tensor([7, 7, 0, 39, 12], dtype=torch.int32).cuda()
    out = QuantRows(torch.full((5, 112), 55, dtype=torch.int8).cuda(), torch.zeros(5).cuda(), 70)       # wider rows than needed
    assert dev.quantize_rows(x, rows=rows, out=out) is out
    want_q, want_s = defined_rows(x.cpu().double().numpy()[[7, 7, 0, 39, 12]])
    got = out.q.cpu().numpy()
    assert np.array_equal(got[:, :70], want_q) and np.array_equal(out.scale.cpu().numpy(), want_s)
    assert not got[:, 70:80].any() and (got[:, 80:] == 55).all()      # the last group is filled up, columns behind it are not touched
    dev.synchronize()
    dev.quantize_rows(x, rows=torch.tensor([-1, 40, 3], dtype=torch.int32).cuda())
    with pytest.raises(IndexError):
        dev.synchronize()
    dev.synchronize()
    assert dev.quantize_rows(torch.zeros(0, 5).cuda()).shape == (0, 5)


# ------------------------------------------------------------------------------------------------------------ product
def product_case(seed, M, N, K, bias=True, full=False):
    rng = np.random.default_rng(seed)
    draw = (lambda r: rng.integers(-128, 128, (r, K))) if full else (lambda r: np.clip(np.rint(rng.normal(0, 40, (r, K))), -127, 127))
    A, B = draw(M).astype(np.int8), draw(N).astype(np.int8)
    sa, sb = np.exp(rng.normal(-3, 1, M)).astype(np.float32), np.exp(rng.normal(-3, 1, N)).astype(np.float32)
    b = rng.normal(0, 1, N).astype(np.float32) if bias else None
    return A, sa, B, sb, b


def check_product(dev, A, sa, B, sb, b, out="f32", into=None):
    K = A.shape[1]
    a, w = quant_rows(A, sa, K), quant_rows(B, sb, K)
    C = torch.full((len(A), len(B)), 9.0, dtype=T[out]).cuda() if into is None else into
    got = dev.matmul_i8(a, w, bias=None if b is None else torch.from_numpy(b).cuda(), out=C)
    assert got is C
    prod = (A.astype(np.float64) @ B.astype(np.float64).T) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)[None, :]
    add = np.zeros(len(B)) if b is None else b.astype(np.float64)
    want = prod + add[None, :]
    # four roundings of the product (conversion, two scales, and as a part of the sum), one of the bias, to first order;
    # then the one to the output's type
    tol = 1.01 * 2.0 ** -24 * (4 * np.abs(prod) + np.abs(add)[None, :])
    if out != "f32":
        tol += HALF[out] * (np.abs(want) + tol) + (2.0 ** -25 if out == "f16" else 0.0)
    d = np.abs(C.double().cpu().numpy() - want)
    bad = np.argwhere(d > tol)
    assert not len(bad), (len(bad), bad[:4], d[tuple(bad[0])], tol[tuple(bad[0])])


SHAPES = [(1, 1, 1), (1, 7, 16), (1, 1682, 20), (2, 33, 31), (3, 5, 64), (5, 300, 65), (16, 16, 128), (17, 100, 100), (31, 129, 127), (33, 257, 256),
          (64, 1000, 1000), (65, 63, 513), (127, 129, 48), (128, 128, 64), (200, 130, 2050), (257, 255, 190), (1, 4099, 4096), (8, 513, 8192), (300, 520, 4000),
          (512, 768, 1024), (40, 40, 20000)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(dev, M, N, K):
    check_product(dev, *product_case(M * 7 + N * 3 + K, M, N, K, bias=(M + N + K) % 2 == 0))


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 512), (77, 503, 1210), (130, 260, 64), (300, 1027, 700), (16, 31, 33)])
def test_product_16_bit_outputs(dev, out, M, N, K):
    A, sa, B, sb, b = product_case(M + N + K, M, N, K)
    sa *= np.float32(0.02)                                    # (half precision ends at 65504)
    check_product(dev, A, sa, B, sb, b, out)


@pytest.mark.parametrize("K", [1, 63, 1040, 1041, 70001, 131071])
def test_product_of_extreme_values_is_exact_in_32_bits(dev, K):
    """All products 128 * 128: the sum reaches 2^31 - 2^14 at the largest K allowed."""
    from tfrec_amd.device import QuantRows
    ld = (K + 15) // 16 * 16
    for M, N in ((1, 3), (20, 3), (130, 140)):
        a = QuantRows(torch.full((M, ld), -128, dtype=torch.int8).cuda(), torch.ones(M).cuda(), K)
        b = QuantRows(torch.full((N, ld), -128, dtype=torch.int8).cuda(), torch.ones(N).cuda(), K)
        C = dev.matmul_i8(a, b, out=torch.zeros(M, N).cuda())
        assert (C.cpu() == float(np.float32(128 * 128 * K))).all()


def test_product_pitches_and_neighbours_untouched(dev):
    """Rows of A, B and C inside wider matrices, C at an odd offset: only the M x N values are written."""
    from tfrec_amd.device import QuantRows
    A, sa, B, sb, b = product_case(11, 70, 45, 90)
    for out in ("f32", "bf16"):
        big = torch.full((72, 61), 3.0, dtype=T[out]).cuda()
        check_product(dev, A, sa, B, sb, b, out, into=big[1:71, 5:50])
        edge = big.clone()
        edge[1:71, 5:50] = 3.0
        assert (edge == 3.0).all()
    wide = torch.from_numpy(np.random.default_rng(0).integers(-127, 128, (70, 160)).astype(np.int8)).cuda()
    wide[:, :90] = torch.from_numpy(A).cuda()
    a = QuantRows(wide, torch.from_numpy(sa).cuda(), 90)
    assert torch.equal(dev.matmul_i8(a, quant_rows(B, sb, 90), out=torch.empty(70, 45).cuda()),
                       dev.matmul_i8(quant_rows(A, sa, 90), quant_rows(B, sb, 90), out=torch.empty(70, 45).cuda()))


def test_product_of_rows_without_a_scale(dev):
    """NaN and zero scales: NaN rows and columns, and zeros."""
    A, sa, B, sb, b = product_case(2, 40, 70, 30)
    sa[3], sa[4], sb[7], sb[8] = np.nan, 0.0, np.nan, 0.0
    C = dev.matmul_i8(quant_rows(A, sa, 30), quant_rows(B, sb, 30), bias=torch.from_numpy(b).cuda(), out=torch.empty(40, 70).cuda()).cpu().numpy()
    assert np.isnan(C[3]).all() and np.isnan(C[:, 7]).all()
    keep = np.ones(70, bool)
    keep[7] = False
    assert np.array_equal(C[4, keep], b[keep]) and (np.delete(C, 3, 0)[:, 8] == b[8]).all()
    assert np.isfinite(np.delete(np.delete(C, 3, 0), 7, 1)).all()


def test_empty_products(dev):
    A, sa, B, sb, b = product_case(2, 3, 4, 5)
    none = quant_rows(np.zeros((0, 5), np.int8), np.zeros(0), 5)
    assert dev.matmul_i8(none, quant_rows(B, sb, 5), out=torch.empty(0, 4).cuda()).shape == (0, 4)
    assert dev.matmul_i8(quant_rows(A, sa, 5), none, out=torch.empty(3, 0).cuda()).shape == (3, 0)


def test_product_beyond_32_bit_offsets(dev):
    """C of more than 2^32 values: the corners are where they belong."""
    from tfrec_amd.device import QuantRows
    M = N = 66000
    g = torch.Generator(device="cuda").manual_seed(1)
    a = QuantRows(torch.randint(-127, 128, (M, 16), generator=g, device="cuda", dtype=torch.int8), torch.ones(M, device="cuda"), 16)
    b = QuantRows(torch.randint(-127, 128, (N, 16), generator=g, device="cuda", dtype=torch.int8), torch.ones(N, device="cuda"), 16)
    C = dev.matmul_i8(a, b, out=torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"))
    for r in (0, 31, 65000, M - 1):
        want = (a.q[r].double()[None, :] @ b.q.double().t())[0]
        assert torch.equal(C[r].double(), want.float().to(torch.bfloat16).double())


# -------------------------------------------------------------------------------------------------------------- top-k
def scores_f32(Pq, sp, Qq, sq, b):
    acc = (Pq.astype(np.float64) @ Qq.astype(np.float64).T).astype(np.float32)       # whole numbers below 2^24
    with np.errstate(all="ignore"):
        return (acc * sp[:, None]) * sq[None, :] + (b if b is not None else np.float32(0))[None, :] if b is not None else (acc * sp[:, None]) * sq[None, :]


def expected_topk(S, k, masks, lo=0, hi=None, id_lo=0):
    """Lists under (score descending, id ascending), NaN and -inf scores left out, -1 / -inf behind the last."""
    n, I = S.shape
    hi = I if hi is None else hi
    ids, sc = np.full((n, k), -1, np.int32), np.full((n, k), -np.inf, np.float32)
    for r in range(n):
        row = S[r].copy()
        if masks is not None:
            row[masks[r]] = -np.inf
        at = np.arange(lo, hi)[(row[lo:hi] > -np.inf)]
        at = at[np.lexsort((at, -row[at].astype(np.float64)))][:k]
        ids[r, :len(at)], sc[r, :len(at)] = at + id_lo, row[at]
    return ids, sc


def topk_case(seed, U, I, d, train=0, spread=1.0, full_rows=()):
    rng = np.random.default_rng(seed)
    row = lambda n: np.clip(np.rint(rng.normal(0, 40, (n, d))), -127, 127).astype(np.int8)       # noqa: E731
    Pq, Qq = row(U), row(I)
    sp, sq = np.exp(rng.normal(-5, spread, U)).astype(np.float32), np.exp(rng.normal(-5, spread, I)).astype(np.float32)
    b = rng.normal(0, 0.1, I).astype(np.float32)
    masks = None
    if train:
        masks = [np.sort(rng.choice(I, min(I, int(rng.integers(0, 2 * train + 1))), replace=False)) for _ in range(U)]
        for u in full_rows:
            masks[u] = np.arange(I)
    return Pq, sp, Qq, sq, b, masks


def csr(masks):
    ptr = np.concatenate([[0], np.cumsum([len(m) for m in masks])]).astype(np.int64)
    idx = np.concatenate([np.asarray(m, np.int32) for m in masks] + [np.zeros(0, np.int32)]).astype(np.int32)
    return torch.from_numpy(ptr).cuda(), torch.from_numpy(np.concatenate([idx, np.zeros(1, np.int32)])).cuda()


def check_topk(dev, case, users, k, lo=0, hi=None, compact=False):
    Pq, sp, Qq, sq, b, masks = case
    d = Pq.shape[1]
    users = np.asarray(users, np.int32)
    hi = len(Qq) if hi is None else hi
    want = expected_topk(scores_f32(Pq[users], sp[users], Qq, sq, b), k, None if masks is None else [masks[u] for u in users], lo, hi)
    P = quant_rows(Pq[users], sp[users], d) if compact else quant_rows(Pq, sp, d)
    ids, sc = dev.score_topk_i8(P, quant_rows(Qq, sq, d), None if b is None else torch.from_numpy(b).cuda(), torch.from_numpy(users).cuda(), k,
                                train=None if masks is None else csr(masks), item_range=(lo, hi), compact=compact)
    dev.synchronize()
    ids, sc = ids.numpy(), sc.numpy()
    for r in np.flatnonzero((ids != want[0]).any(1))[:1]:
        e = int(np.flatnonzero(ids[r] != want[0][r])[0])
        assert False, ("row", int(r), "place", e, ids[r, e:e + 4], want[0][r, e:e + 4], sc[r, e:e + 4], want[1][r, e:e + 4])
    assert np.array_equal(sc, want[1])


@pytest.mark.parametrize("n,I,d,k,train", [
    (1, 1, 1, 1, 0), (1, 40, 5, 50, 0), (1, 63, 16, 10, 3), (2, 65, 17, 7, 5), (3, 700, 20, 50, 30), (1, 5000, 64, 100, 40), (5, 33000, 33, 240, 100),
    (33, 4096, 128, 20, 10), (31, 9999, 100, 113, 700), (64, 20000, 64, 1, 8), (65, 1682, 20, 50, 80), (130, 3001, 256, 112, 20), (300, 6000, 48, 50, 16),
    (943, 1682, 20, 50, 85), (700, 12345, 64, 50, 10), (2100, 5000, 200, 10, 5), (1100, 300, 8, 200, 50), (4, 70000, 250, 64, 1500)])
def test_topk(dev, n, I, d, k, train):
    case = topk_case(n * 31 + I + d + k, n, I, d, train)
    check_topk(dev, case, np.random.default_rng(n).permutation(n), k)


def test_topk_without_bias_and_without_train(dev):
    Pq, sp, Qq, sq, b, masks = topk_case(3, 50, 3000, 24, 0)
    check_topk(dev, (Pq, sp, Qq, sq, None, None), np.arange(50), 30)


@pytest.mark.parametrize("n", [3, 40, 600])
def test_topk_item_ranges_compact_rows_and_repeated_users(dev, n):
    case = topk_case(n, n, 9000, 40, 50)
    users = np.random.default_rng(0).integers(0, n, n + 5)
    for lo, hi in ((0, 9000), (17, 8001), (8999, 9000), (500, 531), (40, 40), (4096, 8192)):
        check_topk(dev, case, users, 20, lo, hi)
    check_topk(dev, case, users, 20, 100, 7000, compact=True)


@pytest.mark.parametrize("n", [2, 50, 700])
def test_topk_rows_that_the_masks_empty_and_nearly_empty(dev, n):
    """Users whose train items are all items, all but one, and all inside the item range."""
    I = 2500
    case = topk_case(4, n, I, 33, 30, full_rows=(0,))
    case[5][1] = np.delete(np.arange(I), 1234)
    if n > 2:
        case[5][2] = np.arange(100, 2400)
        case[5][3] = np.zeros(0, np.int64)
    check_topk(dev, case, np.arange(n), 50)
    check_topk(dev, case, np.arange(n), 200, 100, 2400)


@pytest.mark.parametrize("n", [2, 40, 700])
@pytest.mark.parametrize("kind", ["all_equal", "two_values", "zero_user", "rising", "falling", "huge_scales"])
def test_topk_ties_and_orders(dev, n, kind):
    """Equal scores rank by id whatever path and split they come through; scores that rise with the id keep every list full."""
    I, d = 7000, 32
    Pq, sp, Qq, sq, b, masks = topk_case(8, n, I, d, 20)
    if kind == "all_equal":
        Qq[:], sq[:], b[:] = Qq[0], sq[0], b[0]
    elif kind == "two_values":
        Qq[:], sq[:] = Qq[0], sq[0]
        b[:] = np.where(np.arange(I) % 3 == 1, 0.5, 0.25)
    elif kind == "zero_user":
        sp[:] = 0.0
        b[:] = np.round(b, 1)
    elif kind in ("rising", "falling"):
        Pq[:], Qq[:], sp[:] = 1, 1, 1e-3
        sq[:] = 0.5 + (np.arange(I) if kind == "rising" else I - np.arange(I)) / I
        b[:] = 0.0
    else:
        sq[:] = np.where(np.arange(I) % 11 == 0, 1e30, 1e-30)
        sp[:] = 1e5
        b[:] = 0
    check_topk(dev, (Pq, sp, Qq, sq, b, masks), np.arange(n), 60)


@pytest.mark.parametrize("n", [2, 40, 700])
def test_topk_infinities_and_nan(dev, n):
    """Biases of +-inf, of the lowest float and NaN; items and users without a scale."""
    Pq, sp, Qq, sq, b, masks = topk_case(21, n, 4000, 20, 10)
    rng = np.random.default_rng(1)
    b[rng.choice(4000, 900, replace=False)] = -np.inf
    b[rng.choice(4000, 20, replace=False)] = np.inf
    b[rng.choice(4000, 900, replace=False)] = np.finfo(np.float32).min
    b[rng.choice(4000, 300, replace=False)] = np.nan
    sq[rng.choice(4000, 300, replace=False)] = np.nan
    sq[rng.choice(4000, 300, replace=False)] = 0.0
    sp[1] = np.nan
    check_topk(dev, (Pq, sp, Qq, sq, b, masks), np.arange(n), 100)


def test_topk_user_ids_out_of_range_are_reported(dev):
    Pq, sp, Qq, sq, b, _ = topk_case(5, 10, 500, 16)
    users = torch.tensor([3, -1, 10, 2 ** 30], dtype=torch.int32).cuda()
    ids, _ = dev.score_topk_i8(quant_rows(Pq, sp, 16), quant_rows(Qq, sq, 16), torch.from_numpy(b).cuda(), users, 5)
    with pytest.raises(IndexError):
        dev.synchronize()
    dev.synchronize()
    want, _ = expected_topk(scores_f32(Pq, sp, Qq, sq, b)[[3, 0, 9, 9]], 5, None)
    assert np.array_equal(ids.numpy(), want)


def test_topk_of_no_users(dev):
    Pq, sp, Qq, sq, b, _ = topk_case(5, 10, 500, 16)
    ids, sc = dev.score_topk_i8(quant_rows(Pq, sp, 16), quant_rows(Qq, sq, 16), None, torch.zeros(0, dtype=torch.int32).cuda(), 5,
                                out_ids=torch.zeros(0, 5, dtype=torch.int32).cuda(), out_scores=torch.zeros(0, 5).cuda())
    assert ids.shape == (0, 5)


def test_topk_of_an_item_table_beyond_32_bit_offsets(dev):
    """A table of more than 2^32 bytes whose best rows lie behind that point."""
    from tfrec_amd.device import QuantRows
    I, d, n = 17_000_000, 256, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randint(-3, 4, (1, d), generator=g, device="cuda", dtype=torch.int8).repeat(I, 1)
    best = torch.tensor([I - 1, 16_900_123, 5, 16_777_217], device="cuda")
    P = torch.randint(-127, 128, (n, d), generator=g, device="cuda", dtype=torch.int8)
    q[best] = P[0]
    for m in (1, n):
        ids, _ = dev.score_topk_i8(QuantRows(P, torch.ones(n, device="cuda"), d), QuantRows(q, torch.ones(I, device="cuda"), d), None,
                                   torch.arange(m, dtype=torch.int32, device="cuda"), 4)
        assert list(ids.numpy()[0]) == sorted(best.tolist())


def test_topk_of_more_users_than_one_pass_holds(dev):
    """30000 listed users (20 distinct ones) over 300k items: the table of best scores is cut into passes."""
    case = topk_case(6, 20, 300000, 16, 30)
    users = np.tile(np.arange(20, dtype=np.int32), 1500)
    Pq, sp, Qq, sq, b, masks = case
    for compact in (False, True):
        P = quant_rows(Pq[users], sp[users], 16) if compact else quant_rows(Pq, sp, 16)
        ids, sc = dev.score_topk_i8(P, quant_rows(Qq, sq, 16), torch.from_numpy(b).cuda(), torch.from_numpy(users).cuda(), 10, train=csr(masks),
                                    compact=compact)
        want = expected_topk(scores_f32(Pq, sp, Qq, sq, b), 10, masks)
        assert (ids.numpy().reshape(1500, 20, 10) == want[0][None]).all() and (sc.numpy().reshape(1500, 20, 10) == want[1][None]).all()


# --------------------------------------------------------------------------------------------------------- run together
def test_product_then_dense_topk_equals_the_fused_form(dev):
    """The matrix of matmul_i8 ranked by topk_dense is what score_topk_i8 returns, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(3)
    P, Q = torch.randn(90, 50, generator=g, device="cuda"), torch.randn(4100, 50, generator=g, device="cuda")
    b = torch.randn(4100, generator=g, device="cuda")
    p, q = dev.quantize_rows(P), dev.quantize_rows(Q)
    S = dev.matmul_i8(p, q, bias=b, out=torch.empty(90, 4100, device="cuda"))
    ids, sc = dev.topk_dense(S, 40)
    ids2, sc2 = dev.score_topk_i8(p, q, b, torch.arange(90, dtype=torch.int32, device="cuda"), 40)
    assert np.array_equal(ids.numpy(), ids2.numpy()) and np.array_equal(sc.numpy(), sc2.numpy())


@pytest.mark.parametrize("n,I,d", [(5, 900, 20), (300, 5000, 64), (40, 2000, 256), (3, 40000, 100)])
def test_score_mode_i8_equals_kept_tables(dev, n, I, d):
    """score_topk, its shard form and eval_fullrank in the 8-bit mode against quantised tables that are kept."""
    from tfrec_amd.device import SCORE_I8
    rng = np.random.default_rng(n)
    P, Q, b = rng.normal(0, 0.1, (n, d)).astype(np.float32), rng.normal(0, 0.1, (I, d)).astype(np.float32), rng.normal(0, 0.01, I).astype(np.float32)
    masks = [np.sort(rng.choice(I, 12, replace=False)) for _ in range(n)]
    test = [np.sort(rng.choice(I, 6, replace=False)) for _ in range(n)]
    tr, te = csr(masks), csr(test)
    up = lambda x: torch.from_numpy(x).cuda()       # noqa: E731
    users = rng.permutation(n).astype(np.int32)
    ids, sc = dev.score_topk_i8(dev.quantize_rows(up(P)), dev.quantize_rows(up(Q)), up(b), up(users), 25, train=tr)
    ids, sc = ids.numpy(), sc.numpy()
    a, s = dev.score_topk(up(P), up(Q), up(b), up(users), 25, train=tr, mode=SCORE_I8)
    assert np.array_equal(a.numpy(), ids) and np.array_equal(s.numpy(), sc)
    parts = [dev.score_topk_shard(up(P[users]), up(Q[lo:hi]), up(b[lo:hi]), lo, up(users), 25, train=tr, mode=SCORE_I8) for lo, hi in ((0, I // 3), (I // 3, I), (I, I))]
    gi, gs = np.stack([x[0].numpy() for x in parts]), np.stack([x[1].numpy() for x in parts])
    m, ms = dev.topk_merge(up(gi), up(gs), 3, n, 25)
    assert np.array_equal(m.numpy(), ids) and np.array_equal(ms.numpy(), sc)
    lists = torch.zeros(n, 25, dtype=torch.int32).cuda()
    curves = dev.eval_fullrank(up(P), up(Q), up(b), up(users), tr, te, 25, mode=SCORE_I8, mean_mode=1, out_ids=lists)
    assert np.array_equal(lists.cpu().numpy(), ids)
    hits = np.array([[len(np.intersect1d(ids[r, :j + 1], test[u])) / (j + 1) for j in range(25)] for r, u in enumerate(users)])
    np.testing.assert_allclose(curves[0], hits.mean(0), rtol=1e-5, atol=1e-7)


def test_captured_calls_replay_on_new_inputs(dev):
    """Quantise, product and top-k in one graph: replays on changed inputs, with eager work and a growing workspace between."""
    from tfrec_amd.device import QuantRows
    g = torch.Generator(device="cuda").manual_seed(9)
    M, N, K, k = 20, 3000, 72, 10
    X, W, b = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda"), torch.randn(N, generator=g, device="cuda")
    q = dev.quantize_rows(W)
    a = QuantRows(torch.zeros(M, 80, dtype=torch.int8, device="cuda"), torch.zeros(M, device="cuda"), K)
    C, users = torch.zeros(M, N, device="cuda"), torch.arange(M, dtype=torch.int32, device="cuda")
    ids, sc = torch.zeros(M, k, dtype=torch.int32, device="cuda"), torch.zeros(M, k, device="cuda")

    def step():
        dev.quantize_rows(X, out=a)
        dev.matmul_i8(a, q, bias=b, out=C)
        dev.score_topk_i8(a, q, b, users, k, out_ids=ids, out_scores=sc)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=dev._torch_stream):
        step()
    for i in range(4):
        X.copy_(torch.randn(M, K, generator=g, device="cuda") * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (C, ids, sc)]
        for t in (C, ids, sc):
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, (C, ids, sc)))
        dev.topk_dense(torch.randn(4000 * (i + 1), 64, generator=g, device="cuda"), 5)         # the workspace grows: the graph's block stays
        torch.cuda.synchronize()


# --------------------------------------------------------------------------------------- the sides of the launch rules
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(65, 4099, 256), (500, 1101, 300), (513, 1030, 1000), (1000, 3301, 200), (129, 12700, 20), (2100, 4701, 600), (4100, 2561, 529)])
def test_product_tiles(dev, M, N, K, out):
    A, sa, B, sb, b = product_case(M + N + K, M, N, K, bias=K % 3 != 0)
    check_product(dev, A, sa * np.float32(0.02), B, sb, b, out)


@pytest.mark.parametrize("M,N,K", [(130, 40001, 600), (300, 5003, 777), (20, 30001, 1030), (33, 70000, 520), (129, 41000, 640), (70, 9000, 4097), (128, 8193, 1281)])
def test_product_tiles_of_few_rows(dev, M, N, K):
    check_product(dev, *product_case(M + N + K, M, N, K, bias=M % 2 == 0))


def test_product_of_rows_far_apart(dev):
    """Rows 16 MiB apart: a tile's rows do not fit 32-bit offsets."""
    M, N, K, ld = 66, 9000, 520, 1 << 24
    A, sa, B, sb, b = product_case(7, M, N, K)
    wide = torch.zeros(M, ld, dtype=torch.int8, device="cuda")
    wide[:, :K] = torch.from_numpy(A).cuda()
    from tfrec_amd.device import QuantRows
    a, w, bias = QuantRows(wide, torch.from_numpy(sa).cuda(), K), quant_rows(B, sb, K), torch.from_numpy(b).cuda()
    got, want = (dev.matmul_i8(x, w, bias=bias, out=torch.empty(M, N, device="cuda")) for x in (a, quant_rows(A, sa, K)))
    dev.synchronize()
    assert torch.equal(got, want)


def test_product_tiles_into_a_pitched_slice(dev):
    """Every tile kernel into an output whose rows start off their 16 bytes; what lies around it stays."""
    for M, N, K in ((1000, 3301, 200), (500, 1101, 300), (2100, 4701, 512), (70, 131, 64)):
        A, sa, B, sb, b = product_case(M + K, M, N, K)
        a, w = quant_rows(A, sa, K), quant_rows(B, sb, K)
        for out in ("f32", "bf16"):
            dt = {"f32": torch.float32, "bf16": torch.bfloat16}[out]
            whole = torch.full((M + 2, N + 5), 7.0, dtype=dt, device="cuda")
            dev.matmul_i8(a, w, bias=torch.from_numpy(b).cuda(), out=whole[1:-1, 3:-2])
            want = torch.empty(M, N, dtype=dt, device="cuda")
            dev.matmul_i8(a, w, bias=torch.from_numpy(b).cuda(), out=want)
            dev.synchronize()
            assert torch.equal(whole[1:-1, 3:-2], want)
            whole[1:-1, 3:-2] = 7.0
            assert bool((whole == 7.0).all())


@pytest.mark.parametrize("n,I,d,k,train", [
    (200, 6000, 100, 20, 10), (97, 4097, 128, 33, 5), (20, 8000, 128, 10, 3), (33, 9000, 200, 10, 5), (3, 120000, 64, 20, 30), (300, 120000, 20, 20, 30),
    (40, 110000, 150, 5, 3), (260, 100001, 31, 113, 2), (300, 7000, 192, 20, 9), (30, 5001, 129, 20, 9)])
def test_topk_sets_and_groups(dev, n, I, d, k, train):
    case = topk_case(n + I + d + k, n, I, d, train)
    check_topk(dev, case, np.arange(n)[::-1], k)


@pytest.mark.parametrize("n,I", [(3, 110000), (300, 100000), (70, 5000)])
def test_topk_of_large_groups_with_ties(dev, n, I):
    """Scores that repeat, so that lists end among equals, train items among the best."""
    rng = np.random.default_rng(I)
    Pq, sp, Qq, sq, b, _ = topk_case(n, n, I, 16, 0)
    Qq[:] = Qq[rng.integers(0, 40, I)]
    sq[:] = np.float32(0.5)
    b[:] = np.float32(0.25)
    S = scores_f32(Pq, sp, Qq, sq, b)
    masks = [np.sort(rng.choice(np.flatnonzero(S[u] == S[u].max()), 30, replace=False)) if u % 3 else np.zeros(0, np.int64) for u in range(n)]
    check_topk(dev, (Pq, sp, Qq, sq, b, masks), np.arange(n), 20)


@pytest.mark.parametrize("n,I", [(3, 900), (5, 120000), (200, 20000)])
def test_topk_of_negative_scales(dev, n, I):
    Pq, sp, Qq, sq, b, masks = topk_case(n, n, I, 40, 6)
    rng = np.random.default_rng(1)
    sp *= rng.choice([-1, 1], n).astype(np.float32)
    sq *= rng.choice([-1, 1], I).astype(np.float32)
    b *= np.float32(0.001)
    check_topk(dev, (Pq, sp, Qq, sq, b, masks), np.arange(n), 25)


@pytest.mark.parametrize("n,I", [(2, 100000), (300, 6000)])
def test_captured_topk_with_scratch(dev, n, I):
    """Two graphs of calls that take scratch: replays in turn on changed inputs, eager calls that need more scratch between."""
    g = torch.Generator(device="cuda").manual_seed(n)
    P = torch.randn(n, 48, generator=g, device="cuda")
    Q = torch.randn(I, 48, generator=g, device="cuda")
    p, q = dev.quantize_rows(P), dev.quantize_rows(Q)
    users = torch.arange(n, dtype=torch.int32, device="cuda")
    outs = [(torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")) for k in (7, 30)]

    def step(i):
        dev.score_topk_i8(p, q, None, users, (7, 30)[i], out_ids=outs[i][0], out_scores=outs[i][1])
    step(0), step(1)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=dev._torch_stream):
            step(i)
    for turn in range(3):
        dev.quantize_rows(torch.randn(n, 48, generator=g, device="cuda"), out=p)
        torch.cuda.synchronize()
        for i in (0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [t.clone() for o in outs for t in o]
        for o in outs:
            o[0].zero_(), o[1].zero_()
        step(0), step(1)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, [t for o in outs for t in o]))
        big = torch.randint(-127, 128, (5000 * (turn + 1), 64), dtype=torch.int8, device="cuda")
        wide = quant_rows(big.cpu().numpy(), np.ones(len(big), np.float32), 64)
        dev.score_topk_i8(wide, wide, None, torch.arange(600 * (turn + 1), dtype=torch.int32, device="cuda"), 10)
        torch.cuda.synchronize()


def test_freed_rows_are_refused_and_an_empty_train_matrix_masks_nothing(dev):
    from tfrec_amd.device import QuantRows
    rng = np.random.default_rng(4)
    P, Q = rng.normal(0, 1, (3, 20)).astype(np.float32), rng.normal(0, 1, (50, 20)).astype(np.float32)
    p, q = dev.quantize_rows(torch.from_numpy(P).cuda()), dev.quantize_rows(torch.from_numpy(Q).cuda())
    users = torch.arange(3, dtype=torch.int32).cuda()
    empty = torch.zeros(4, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    want = dev.score_topk_i8(p, q, None, users, 5)
    got = dev.score_topk_i8(p, q, None, users, 5, train=empty)
    dev.synchronize()
    assert np.array_equal(want[0].numpy(), got[0].numpy()) and np.array_equal(want[1].numpy(), got[1].numpy())
    q.q.free()
    with pytest.raises(ValueError):
        dev.matmul_i8(p, q)
    with pytest.raises(ValueError):
        dev.score_topk_i8(p, q, None, users, 5)
    with pytest.raises(ValueError):
        QuantRows(torch.zeros(4, 64, dtype=torch.int8).cuda()[:, :32], torch.zeros(4).cuda(), 30)


def test_two_contexts_on_their_own_streams(dev):
    """Calls of two contexts that overlap: each has scratch of its own."""
    from tfrec_amd.device import Device
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    devs = [Device(0, s.cuda_stream) for s in streams]
    cases = [topk_case(50 + i, 300, 20000, 40, 8) for i in range(2)]
    held, want = [], []
    for Pq, sp, Qq, sq, b, masks in cases:
        held.append((quant_rows(Pq, sp, 40), quant_rows(Qq, sq, 40), torch.from_numpy(b).cuda(), torch.arange(300, dtype=torch.int32).cuda(), csr(masks)))
        want.append(expected_topk(scores_f32(Pq, sp, Qq, sq, b), 20, masks))
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for i, d in enumerate(devs):
            p, q, b, users, train = held[i]
            got.append((i, d.score_topk_i8(p, q, b, users, 20, train=train), d.matmul_i8(p, q, bias=b)))
    for d in devs:
        d.synchronize()
    for i, (ids, sc), C in got:
        assert np.array_equal(ids.numpy(), want[i][0]) and np.array_equal(sc.numpy(), want[i][1])
        assert np.array_equal(C.numpy()[:2], scores_f32(*cases[i][:5])[:2])
    del got, C, ids, sc
    for d in devs:
        d.close()
