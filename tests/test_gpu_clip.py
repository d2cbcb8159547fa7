"""Gradient norm and clipping on the GPU against their definition in 64 bits, the gradients of the BPR loss against the
formula's and against differences, and models trained with a bounded step."""
import numpy as np
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


T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def expect(host, max_norm):
    """(norm, scale) in double; the bound is what the entry point is handed, a float32."""
    max_norm = float(np.float32(max_norm))
    total = float(sum(np.sum(np.square(x.double().numpy().reshape(-1))) for x in host))
    norm = float(np.sqrt(total))
    return norm, max_norm / max(norm, max_norm)


def close(got, x, s, exact=False):
    """got = x * s: the scale and the product round to float32 (half a step each), then the product to the type."""
    want = x.double() * s
    if exact:
        assert torch.equal(got.cpu(), x)
        return
    tol = want.abs() * (2 * 2.0 ** -24 + (STEP[x.dtype] if x.dtype != torch.float32 else 0)) * 1.01 + TINY[x.dtype] / 2 + 2.0 ** -149
    assert ((got.cpu().double() - want).abs() <= tol).all()


def run_clip(dev, host, max_norm, in_place):
    grads = [x.cuda() for x in host]
    out = None if in_place else [torch.full_like(x, 5.0) for x in grads]
    norm = dev.clip_grads(grads, max_norm, out=out, norm=torch.zeros(1).cuda())
    want_norm, s = expect(host, max_norm)
    assert abs(float(norm) - want_norm) <= 2.0 ** -23 * want_norm
    for g, x in zip(grads if in_place else out, host):
        close(g, x, s, exact=want_norm <= max_norm)
    if not in_place:
        assert all(torch.equal(g.cpu(), x) for g, x in zip(grads, host))
    # a kept list gives the same
    again = [x.cuda() for x in host]
    lst = dev.grad_list(again, out=None if in_place else [torch.full_like(x, 5.0) for x in again])
    n2 = dev.grad_norm(lst, norm=torch.zeros(1).cuda())
    n3 = dev.clip_grads(lst, max_norm, norm=torch.zeros(1).cuda())
    assert abs(float(n2) - want_norm) <= 2.0 ** -23 * want_norm and abs(float(n3) - want_norm) <= 2.0 ** -23 * want_norm
    for g, x in zip(lst.out, host):
        close(g, x, s, exact=want_norm <= max_norm)
    assert float(dev.grad_norm(grads if not in_place else [x.cuda() for x in host], norm=torch.zeros(1).cuda())) == float(norm)


LENGTHS = [[1], [0], [60000, 5000], [8192 * 8], [8192 * 8 + 1], [9000, 9000, 9000, 1], [0, 3, 0], [17], [255, 1, 4096], [8191], [8192], [8193, 8192, 1], [100003], [7] * 95, [11] * 96, [5] * 97, [3, 20000] * 150, [3_000_001, 2, 50]]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_clip_lengths(dev, lengths, in_place):
    g = torch.Generator().manual_seed(sum(lengths))
    types = [list(T.values())[i % 3] for i in range(len(lengths))]
    host = [(torch.randn(n, generator=g) * 0.1).to(t) for n, t in zip(lengths, types)]
    norm = expect(host, 1.0)[0]
    for bound in (0.37 * norm + 1e-3, 1.5 * norm + 1.0):
        run_clip(dev, host, bound, in_place)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_clip_tensors_at_any_alignment(dev, dtype):
    """Slices of one buffer that begin at every offset of a 16-byte line, sources and outputs shifted against each other."""
    g = torch.Generator().manual_seed(4)
    flat = torch.randn(400000, generator=g).to(T[dtype]).cuda()
    to = torch.full((400100,), 2.0, dtype=T[dtype]).cuda()
    grads, out, at = [], [], 0
    for i, n in enumerate([9001, 8192, 16385, 1, 40000, 8193, 2, 30001] * 2):
        grads.append(flat[at:at + n])
        out.append(to[at + 3 + i:at + 3 + i + n])
        at += n + i
    norm = dev.clip_grads(grads, 7.5, out=out, norm=torch.zeros(1).cuda())
    host = [x.cpu() for x in grads]
    want, s = expect(host, 7.5)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    untouched = torch.ones_like(to, dtype=torch.bool)
    at = 0
    for i, (o, x) in enumerate(zip(out, host)):
        close(o, x, s)
        untouched[at + 3 + i:at + 3 + i + x.numel()] = False
        at += x.numel() + i
    assert (to[untouched] == 2.0).all()


def test_clip_extreme_values(dev):
    """Squares that float32 could not hold, subnormal values, a zero gradient."""
    for vals in ([3e38, -2e38, 1e-30], [1e-44, 3e-45, -1e-40], [1e-20] * 5, [0.0] * 9, [-0.0, 0.0]):
        host = [torch.tensor(vals, dtype=torch.float32)]
        want, s = expect(host, 0.5)
        grads = [host[0].cuda()]
        norm = dev.clip_grads(grads, 0.5, norm=torch.zeros(1).cuda())
        if want < 3.4e38:
            assert abs(float(norm) - want) <= 2.0 ** -23 * want + 2.0 ** -149
        else:
            assert float(norm) == np.inf                    # the norm itself leaves float32; the scale does not
        close(grads[0], host[0], s)


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_spoils_every_value(dev, bad):
    grads = [torch.randn(5000).cuda(), torch.randn(3).to(torch.bfloat16).cuda(), torch.zeros(70, dtype=torch.float16).cuda()]
    grads[0][4321] = bad
    norm = dev.clip_grads(grads, 1.0, norm=torch.zeros(1).cuda())
    assert not np.isfinite(float(norm))
    assert all(torch.isnan(g).all() for g in grads)


def test_norm_counts_a_repeated_tensor_twice_and_clip_refuses_it(dev):
    x = torch.randn(1000).cuda()
    one, two = float(dev.grad_norm([x], norm=torch.zeros(1).cuda())), float(dev.grad_norm([x, x], norm=torch.zeros(1).cuda()))
    assert abs(two - one * np.sqrt(2)) < 1e-5 * two
    with pytest.raises(ValueError, match="overlaps"):
        dev.clip_grads([x, x], 1.0)
    with pytest.raises(ValueError, match="overlaps"):
        dev.clip_grads([x[:600], x[500:]], 1.0)
    y = torch.zeros(2000).cuda()
    dev.clip_grads([x, x], 1.0, out=[y[:1000], y[1000:]])    # read twice, written apart: allowed
    assert torch.equal(y[:1000], y[1000:])


def test_results_repeat_bit_for_bit_and_lists_are_kept(dev):
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(n, generator=g, device="cuda") for n in (100000, 3, 77777)]
    out = [torch.empty_like(x) for x in xs]
    lst = dev.grad_list(xs, out=out)
    norms = [float(dev.clip_grads(lst, 2.0, norm=torch.zeros(1).cuda())) for _ in range(5)]
    first = [o.clone() for o in out]
    assert len(set(norms)) == 1
    dev.clip_grads(lst, 2.0)
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    with pytest.raises(ValueError):
        dev.clip_grads(lst, 2.0, out=out)


def test_clip_beyond_32_bit_offsets(dev):
    n = (1 << 31) + 12345
    x = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    norm = dev.clip_grads([x], 1.0, norm=torch.zeros(1).cuda())
    want = 0.5 * np.sqrt(n)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    v = torch.tensor(0.5 / want, dtype=torch.float32).to(torch.bfloat16)
    assert (x[:5] == v.cuda()).all() and (x[-5:] == v.cuda()).all() and (x[(1 << 31) - 3:(1 << 31) + 3] == v.cuda()).all()
    assert torch.equal(x.min(), x.max())


def test_captured_clip_replays_on_new_gradients(dev):
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [torch.zeros(n, device="cuda") for n in (50000, 7, 8200)]
    out = [torch.zeros_like(x) for x in xs]
    norm = torch.zeros(1, device="cuda")
    lst = dev.grad_list(xs, out=out)
    dev.clip_grads(lst, 1.0, norm=norm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=dev._torch_stream):
        dev.clip_grads(lst, 1.0, norm=norm)
    for i in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda") * 10.0 ** (1 - i))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out] + [norm.clone()]
        dev.clip_grads(lst, 1.0, norm=norm)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, out + [norm]))


# ------------------------------------------------------------------------------------------------- gradients of the loss
def bpr_loss(P, Q, b, u, i, j, reg):
    x = (P[u] * (Q[i] - Q[j])).sum(1) + b[i] - b[j]
    l2 = sum((t * t).sum() / 2 for t in (P[u], Q[i], Q[j], b[i], b[j]))
    return torch.nn.functional.softplus(-(x + 1e-7)).sum() + reg * l2, l2


@pytest.mark.parametrize("U,I,d,B", [(5, 7, 3, 1), (30, 40, 20, 500), (200, 100, 64, 3000), (50, 60, 10, 70), (1000, 900, 128, 4000), (20, 30, 256, 300),
                                     (40, 50, 64, 150000), (7, 9, 20, 0)])
def test_bpr_grads(dev, U, I, d, B):
    rng = np.random.default_rng(U + d + B)
    P, Q, b = [torch.from_numpy(rng.uniform(-0.3, 0.3, s).astype(np.float32)) for s in ((U, d), (I, d), (I,))]
    u, i, j = [torch.from_numpy(rng.integers(0, n, B).astype(np.int32)) for n in (U, I, I)]
    reg = 0.05
    gpu = [t.cuda() for t in (P, Q, b, u, i, j)]
    G = [torch.full_like(t, 7.0) for t in gpu[:3]]
    loss = torch.zeros(2, dtype=torch.float64).cuda()
    dev.bpr_grads(*gpu, reg, *G, loss=loss)
    dev.synchronize()
    assert all(torch.equal(a.cpu(), c) for a, c in zip(gpu[:3], (P, Q, b)))          # parameters stay
    leaves = [t.double().requires_grad_() for t in (P, Q, b)]
    total, l2 = bpr_loss(*leaves, u.long(), i.long(), j.long(), reg)
    want = torch.autograd.grad(total, leaves)
    most = max(1, int(np.bincount(np.concatenate([i.numpy(), j.numpy()])).max()) if B else 1, int(np.bincount(u.numpy()).max()) if B else 1)
    for g, w in zip(G, want):
        # a row's gradient is a sum of up to `most` terms below 1 in size, each a few roundings off; sums in float32
        tol = 2.0 ** -23 * (12 * np.sqrt(most) + 8) * max(1.0, float(w.abs().max()))
        assert float((g.cpu().double() - w).abs().max()) <= tol, (float((g.cpu().double() - w).abs().max()), tol)
    if B:
        assert abs(float(loss[0]) - float((total - reg * l2).detach())) <= 1e-5 * abs(float(total.detach())) and abs(float(loss[1]) - float(l2.detach())) <= 1e-5 * float(l2.detach())
    # the step is the parameters plus -lr times these gradients, bit for bit
    a, c = [t.clone() for t in gpu[:3]], [t.clone() for t in gpu[:3]]
    dev.bpr_sgd_step(*a, *gpu[3:], 0.02, reg)
    for t, g in zip(c, G):
        dev.axpy(t, g, -0.02, n=t.numel())
    dev.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_bpr_grads_against_differences(dev):
    """Directional differences of the float64 loss, at step 1e-6, along random directions."""
    rng = np.random.default_rng(0)
    P, Q, b = [torch.from_numpy(rng.uniform(-0.5, 0.5, s).astype(np.float32)) for s in ((9, 6), (11, 6), (11,))]
    u, i, j = [torch.from_numpy(rng.integers(0, n, 40).astype(np.int32)) for n in (9, 11, 11)]
    G = [torch.empty_like(t).cuda() for t in (P, Q, b)]
    dev.bpr_grads(P.cuda(), Q.cuda(), b.cuda(), u.cuda(), i.cuda(), j.cuda(), 0.1, *G)
    for _ in range(5):
        D = [torch.from_numpy(rng.normal(0, 1, t.shape)) for t in (P, Q, b)]
        f = lambda h: float(bpr_loss(*[t.double() + h * x for t, x in zip((P, Q, b), D)], u.long(), i.long(), j.long(), 0.1)[0])       # noqa: E731
        want = (f(1e-6) - f(-1e-6)) / 2e-6
        got = sum(float((g.cpu().double() * x).sum()) for g, x in zip(G, D))
        assert abs(got - want) <= 1e-5 * (abs(want) + 10)


def test_bpr_grads_refusals(dev):
    P, Q, b = torch.zeros(4, 8).cuda(), torch.zeros(5, 8).cuda(), torch.zeros(5).cuda()
    e = torch.zeros(1, dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="parameters"):
        dev.bpr_grads(P, Q, b, e, e, e, 0.0, P, torch.zeros_like(Q), torch.zeros_like(b))
    with pytest.raises(ValueError, match="shapes"):
        dev.bpr_grads(P, Q, b, e, e, e, 0.0, torch.zeros(3, 8).cuda(), torch.zeros_like(Q), torch.zeros_like(b))


# ------------------------------------------------------------------------------------------------------------- models
class _Data:
    def __init__(self, train, test):
        self.train_matrix, self.test_matrix = train, test


class _Log:
    def __init__(self):
        self.lines = []

    def info(self, s):
        self.lines.append(s)


def small_data():
    import scipy.sparse as sp
    rng = np.random.default_rng(5)
    dense = rng.random((60, 90))
    return _Data(sp.csr_matrix((dense < 0.1).astype(np.float32)), sp.csr_matrix(((dense > 0.1) & (dense < 0.15)).astype(np.float32)))


def make_model(name, data, evaluator, **more):
    from tfrec_amd.device import Device
    from tfrec_amd.model.BPR import BPR
    from tfrec_amd.model.DNSBPR import DNSBPR
    cls = {"BPR": BPR, "DNSBPR": DNSBPR}[name]
    cls.logger = _Log()
    config = dict(factors_num=12, lr=0.05, reg=0.01, epochs=2, batch_size=64, neg_num=4, data_name="t", **more)
    return cls(Device(0), config, data, evaluator)


@pytest.mark.parametrize("name", ["BPR", "DNSBPR"])
@pytest.mark.parametrize("sampler", ["host", "device"])
def test_a_bound_that_no_batch_reaches_changes_nothing(name, sampler, tmp_path, monkeypatch):
    from tfrec_amd.evaluator import FoldOutEvaluator
    monkeypatch.chdir(tmp_path)                 # (DNSBPR leaves its parameters in a file)
    data, tables = small_data(), []
    for bound in (0, 1e6):
        np.random.seed(11)
        m = make_model(name, data, FoldOutEvaluator(data.train_matrix, data.test_matrix, top_k=10), sampler=sampler, clip_norm=bound)
        m.train_model()
        tables.append(m.parameters())
    assert all(np.array_equal(a, b) for a, b in zip(*tables))


def test_clipped_steps_and_8_bit_evaluation_run_together(tmp_path, monkeypatch):
    """A model trained under a bound that every batch reaches, evaluated with 8-bit scores: the tables against the same steps
    in float64, the lists behind the metrics against the definition of the scores."""
    from tfrec_amd.evaluator import FoldOutEvaluator
    data = small_data()
    bound = 0.25
    ev = FoldOutEvaluator.from_config({"score_dtype": "i8", "top_k": 10}, data.train_matrix, data.test_matrix)
    m = make_model("BPR", data, ev, clip_norm=bound, sampler="device")
    P, Q, b = [torch.from_numpy(x).double() for x in m.parameters()]
    users, pos, neg = [torch.from_numpy(x.numpy()).long().reshape(-1) for x in m._device_epoch(0)]
    m._train_epoch_on_device(0)
    n, clipped = m._device_sampler.nnz, 0
    for lo in range(0, n, 64):
        leaves = [t.clone().requires_grad_() for t in (P, Q, b)]
        s = slice(lo, min(lo + 64, n))
        grads = torch.autograd.grad(bpr_loss(*leaves, users[s], pos[s], neg[s], 0.01)[0], leaves)
        norm = float(torch.sqrt(sum((g * g).sum() for g in grads)))
        clipped += norm > bound
        P, Q, b = [t - 0.05 * g * (bound / max(norm, bound)) for t, g in zip((P, Q, b), grads)]
    assert clipped == (n + 63) // 64
    got = m.parameters()
    # every step moves a value by at most 0.05 * 0.25, in float32 arithmetic of a few roundings; so do the steps before it
    for g, w in zip(got, (P, Q, b)):
        assert float(np.abs(g - w.numpy()).max()) <= (n // 64 + 1) * 0.05 * bound * 2.0 ** -20
    curves = ev.evaluate(m).reshape(5, 10)
    scores = m.mf.all_logits(score_dtype="i8")
    hits = []
    for u in range(60):
        test = data.test_matrix[u].indices
        if len(test):
            row = scores[u].copy()
            row[data.train_matrix[u].indices] = -np.inf
            top = np.lexsort((np.arange(90), -row))[:10]
            hits.append([np.isin(top[:j + 1], test).mean() for j in range(10)])
    np.testing.assert_allclose(curves[0], np.mean(hits, 0), rtol=1e-5)
    near = np.abs(m.mf.all_logits() - scores).max()
    # half a step of either row on every product: |p| |q| d / 254 each way
    assert near <= 12 * 2 * np.abs(got[0]).max() * np.abs(got[1]).max() / 254 * 1.01 + 1e-6
    assert np.array_equal(m.mf.all_logits([5, 3, 5], score_dtype="i8"), scores[[5, 3, 5]])


def test_clip_norm_of_sharded_and_adversarial_models_is_refused():
    from tfrec_amd.evaluator import FoldOutEvaluator
    data = small_data()
    ev = FoldOutEvaluator(data.train_matrix, data.test_matrix, top_k=5)
    with pytest.raises(ValueError, match="single-GPU"):
        make_model("BPR", data, ev, clip_norm=1.0, force_sharded=True)


def test_a_list_is_not_made_under_capture(dev):
    xs = [torch.ones(50000, device="cuda"), torch.ones(9000, device="cuda")]
    norm = torch.zeros(1, device="cuda")
    lst = dev.grad_list(xs)
    dev.grad_norm(lst, norm=norm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=dev._torch_stream):
        with pytest.raises(ValueError):
            dev.grad_list(xs)
        dev.grad_norm(lst, norm=norm)
    for v in (2.0, 3.0):
        for x in xs:
            x.fill_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - v * 59000 ** 0.5) <= 2.0 ** -23 * float(norm)
