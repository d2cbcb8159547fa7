"""The 8-bit entry points on outputs that overlap what they read: refused, and nothing is written; rows that lie between each
other's are taken."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from tfrec_amd.sharded import make_device
    before = torch.cuda.current_stream()
    d = make_device(0)
    yield d
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    d.close()


def rows(n, d, seed):
    from tfrec_amd.device import QuantRows
    g = torch.Generator(device="cuda").manual_seed(seed)
    return QuantRows(torch.randint(-127, 128, (n, (d + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8),
                     torch.rand(n, generator=g, device="cuda") + 0.5, d)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_a_product_into_what_it_reads_is_refused(dev, out):
    from tfrec_amd.device import QuantRows
    M, N, K = 64, 32, 128
    buf = torch.zeros(1 << 18, dtype=torch.uint8, device="cuda")
    size = torch.empty(0, dtype=out).element_size()
    C = buf[65536:65536 + M * N * size].view(out).view(M, N)
    end = 65536 + M * N * size
    a, b, bias = rows(M, K, 1), rows(N, K, 2), torch.zeros(N, device="cuda")
    i8 = lambda at, n: buf[at:at + n * K].view(torch.int8).view(n, K)              # noqa: E731
    f4 = lambda at, n: buf[at:at + 4 * n].view(torch.float32)                      # noqa: E731
    for at in (65536, end - 16, 65536 - K * N + 16):
        with pytest.raises(ValueError, match="overlaps"):
            dev.matmul_i8(QuantRows(i8(at, M), a.scale, K), b, out=C)
        with pytest.raises(ValueError, match="overlaps"):
            dev.matmul_i8(a, QuantRows(i8(at, N), b.scale, K), out=C)
    for at in (65536, end - 4):
        with pytest.raises(ValueError, match="overlaps"):
            dev.matmul_i8(QuantRows(a.q, f4(at, M), K), b, out=C)
        with pytest.raises(ValueError, match="overlaps"):
            dev.matmul_i8(a, QuantRows(b.q, f4(at, N), K), out=C)
        with pytest.raises(ValueError, match="overlaps"):
            dev.matmul_i8(a, b, bias=f4(at, N), out=C)
    dev.synchronize()
    assert not buf.any()
    # right behind C, right before it: taken
    want = dev.matmul_i8(a, b, bias=bias, out=torch.empty(M, N, dtype=out, device="cuda")).clone()
    i8(end, M).copy_(a.q)
    f4(65536 - 4 * N, N).copy_(bias)
    dev.matmul_i8(QuantRows(i8(end, M), a.scale, K), b, bias=f4(65536 - 4 * N, N), out=C)
    dev.synchronize()
    assert torch.equal(C, want)


def test_scales_beside_the_rows_of_an_output_are_taken(dev):
    """One matrix holds C, and in the columns behind it, row by row, nothing that a call reads: a bias in one such row's rest."""
    M, N, K = 40, 24, 48
    a, b = rows(M, K, 3), rows(N, K, 4)
    wide = torch.zeros(M, 64, device="cuda")
    bias = wide[7, 30:30 + N]
    bias.copy_(torch.arange(N, device="cuda"))
    want = dev.matmul_i8(a, b, bias=bias.clone(), out=torch.empty(M, N, device="cuda"))
    dev.matmul_i8(a, b, bias=bias, out=wide[:, :N])
    dev.synchronize()
    assert torch.equal(wide[:, :N], want)
    with pytest.raises(ValueError, match="overlaps"):
        dev.matmul_i8(a, b, bias=wide[7, 20:20 + N], out=wide[:, :N])


def test_rows_quantised_onto_what_they_are_made_of_are_refused(dev):
    from tfrec_amd.device import QuantRows
    n, d = 20, 64
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    X = buf[4096:4096 + n * d * 4].view(torch.float32).view(n, d)
    ids = buf[32768:32768 + 4 * n].view(torch.int32)
    q, s = torch.zeros(n, d, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    in_buf = lambda at: buf[at:at + n * d].view(torch.int8).view(n, d)             # noqa: E731
    s_in = lambda at: buf[at:at + 4 * n].view(torch.float32)                       # noqa: E731
    for out in (QuantRows(in_buf(4096), s, d), QuantRows(in_buf(4096 + n * d * 4 - 16), s, d), QuantRows(q, s_in(4096 + 4), d), QuantRows(in_buf(4096 - n * d + 16), s, d)):
        with pytest.raises(ValueError, match="overlaps"):
            dev.quantize_rows(X, out=out)
    for out in (QuantRows(in_buf(32768), s, d), QuantRows(q, s_in(32768 + 4 * n - 4), d)):
        with pytest.raises(ValueError, match="overlaps"):
            dev.quantize_rows(X, rows=ids, out=out)
    with pytest.raises(ValueError, match="overlap"):
        dev.quantize_rows(X, out=QuantRows(in_buf(16384), s_in(16384 + n * d - 4), d))
    dev.synchronize()
    assert not buf.any() and not q.any() and not s.any()
    dev.quantize_rows(X, rows=ids, out=QuantRows(in_buf(4096 + n * d * 4), s_in(32768 + 4 * n), d))         # right behind: taken
    # only the rows that are read count: the last row of X is not among the first n - 1
    dev.quantize_rows(X[:n - 1], out=QuantRows(buf[4096 + (n - 1) * d * 4:][:(n - 1) * d].view(torch.int8).view(n - 1, d), s[:n - 1], d))
    dev.synchronize()


@pytest.mark.parametrize("n,I,k", [(2, 60000, 50), (300, 40000, 20), (2, 60000, 200)])
def test_lists_of_users_whose_train_items_leave_no_cut(dev, n, I, k):
    """Thousands of train items: hardly a slice of the items, or none, is without one, so that the cut of the second step is loose or
    missing and most cells are scored; train items are among the best."""
    import numpy as np
    from test_gpu_int8 import check_topk, scores_f32, topk_case
    Pq, sp, Qq, sq, b, masks = topk_case(I + n + k, n, I, 48, 10)
    rng = np.random.default_rng(n)
    best = np.argsort(-scores_f32(Pq[1:2], sp[1:2], Qq, sq, b)[0])
    masks[0] = np.sort(rng.choice(I, 9000, replace=False))
    masks[1] = np.sort(np.concatenate([best[:2500], rng.choice(best[2500:], 2500, replace=False)]))
    if n > 2:
        masks[2], masks[n - 1] = np.arange(0, I, 3), np.sort(rng.choice(I, 3000, replace=False))
    check_topk(dev, (Pq, sp, Qq, sq, b, masks), np.arange(n), k)
