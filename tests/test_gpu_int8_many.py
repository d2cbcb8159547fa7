"""8-bit calls of more rows and users than one launch may have threads for (2^32 of them): they are launched in pieces, and the
rows on either side of the pieces' borders are what they are elsewhere."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

PIECE = 1 << 22          # workgroups of a launch


@pytest.fixture(scope="module")
def dev():
    from tfrec_amd.sharded import make_device
    before = torch.cuda.current_stream()
    d = make_device(0)
    yield d
    torch.cuda.synchronize()
    torch.cuda.set_stream(before)
    d.close()


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def rows(n, d, seed):
    from tfrec_amd.device import QuantRows
    g = torch.Generator(device="cuda").manual_seed(seed)
    return QuantRows(torch.randint(-127, 128, (n, (d + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8),
                     torch.rand(n, generator=g, device="cuda") * 0.01 + 0.001, d)


@pytest.mark.parametrize("compact", [False, True])
def test_topk_of_few_items_for_more_users_than_a_launch_holds(dev, compact):
    """2^24 + 37 listed users of 64 distinct ones (256 threads a user: beyond 2^32), as table rows and as rows in list order."""
    from tfrec_amd.device import QuantRows
    n, I, d, k, U = (1 << 24) + 37, 70, 16, 2, 64
    p, q = rows(U, d, 1), rows(I, d, 2)
    b = torch.rand(I, device="cuda")
    train = (torch.arange(0, 3 * U + 1, 3, device="cuda"), (torch.arange(3 * U, device="cuda", dtype=torch.int32) % 3) * 20)
    users = torch.arange(n, device="cuda", dtype=torch.int32) % U
    want = dev.score_topk_i8(p, q, b, torch.arange(U, device="cuda", dtype=torch.int32), k, train=train,
                             out_ids=torch.zeros(U, k, dtype=torch.int32, device="cuda"), out_scores=torch.zeros(U, k, device="cuda"))
    P = QuantRows(p.q[users.long()], p.scale[users.long()], d) if compact else p
    ids, sc = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")
    dev.score_topk_i8(P, q, b, users, k, train=train, compact=compact, out_ids=ids, out_scores=sc)
    dev.synchronize()
    assert bool((want[1] > 0).all())
    at = users.long()
    assert torch.equal(ids, want[0][at]) and torch.equal(sc, want[1][at])


def test_no_items_for_more_places_than_a_launch_holds(dev):
    n, k = 18_000_000, 240
    p, q = rows(3, 16, 1), rows(5, 16, 2)
    ids, sc = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")
    dev.score_topk_i8(p, q, None, torch.zeros(n, dtype=torch.int32, device="cuda"), k, item_range=(2, 2), out_ids=ids, out_scores=sc)
    dev.synchronize()
    assert int(ids.max()) == int(ids.min()) == -1 and float(sc.max()) == -np.inf


@pytest.mark.parametrize("listed", [True, False])
def test_more_long_rows_than_a_launch_holds(dev, listed):
    """A workgroup a row: listed rows of a small table beyond 2^32 threads, and a table of its own across a border of the pieces."""
    from tfrec_amd.device import QuantRows
    d = 1030
    g = torch.Generator(device="cuda").manual_seed(3)
    if listed:
        n = (1 << 24) + 3
        X = torch.randn(5, d, generator=g, device="cuda")
        ids = torch.arange(n, device="cuda", dtype=torch.int32) % 5
    else:
        n = PIECE + 11
        X = torch.randn(n, d, generator=g, device="cuda", dtype=torch.bfloat16)
        ids = None
    out = QuantRows(torch.empty(n, 1040, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda"), d)
    dev.quantize_rows(X, rows=ids, out=out)
    dev.synchronize()
    if listed:
        want = dev.quantize_rows(X, out=QuantRows(torch.empty(5, 1040, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda"), d))
        for at in (0, PIECE - 2, PIECE, 2 * PIECE - 1, 4 * PIECE - 3, n - 5):
            sel = ids[at:at + 5].long()
            assert torch.equal(out.q[at:at + 5], want.q[sel]) and torch.equal(out.scale[at:at + 5], want.scale[sel])
        assert torch.equal(out.scale, want.scale[ids.long()])
    else:
        for at in (0, PIECE - 3, n - 6):
            want = dev.quantize_rows(X[at:at + 6].contiguous(), out=QuantRows(torch.empty(6, 1040, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda"), d))
            dev.synchronize()
            assert torch.equal(out.q[at:at + 6], want.q) and torch.equal(out.scale[at:at + 6], want.scale)


@pytest.mark.parametrize("M,N", [(1, (1 << 30) + 5), (3, (1 << 26) + 70), ((1 << 26) + 70, 2)])
def test_products_of_more_rows_than_a_launch_holds(dev, M, N):
    """16 columns; rows of B beyond 2^32 threads, and either operand across a border of the pieces."""
    from tfrec_amd.device import QuantRows
    a, b = rows(min(M, 4096), 16, 1), rows(min(N, 4096), 16, 2)

    def tiled(r, n):
        if n <= 4096:
            return r
        m = (n + 4095) // 4096
        return QuantRows(r.q.repeat(m, 1)[:n], r.scale.repeat(m)[:n], 16)
    A, B = tiled(a, M), tiled(b, N)
    bias = torch.arange(N, device="cuda", dtype=torch.float32) if M < 4 else None
    C = torch.empty(M, N, device="cuda")
    dev.matmul_i8(A, B, bias=bias, out=C)
    # the scores of the distinct rows, each step rounded as the definition has it
    want = (a.q.float() @ b.q.float().t()) * a.scale[:, None] * b.scale[None, :]
    dev.synchronize()
    step = 1 << 26
    for at in range(0, max(M, N), step):
        hi = min(at + step, max(M, N))
        part = torch.arange(at, hi, device="cuda") % 4096
        w = want[:, part] + bias[at:hi] if M < N else want[part]
        assert torch.equal(C[:, at:hi] if M < N else C[at:hi], w)
