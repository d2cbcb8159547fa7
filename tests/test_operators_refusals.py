"""Refusals of the 8-bit and gradient-norm entry points: arguments are checked before a context is entered, so all of this
runs without a GPU (the context is null; a call whose arguments are in order is then refused for the context)."""
import ctypes as C

import numpy as np
import pytest

from tfrec_amd import _lib

A16 = 1 << 20            # an address that is aligned and never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, rc, code, *words):
    assert rc == code, (rc, lib.tfrec_last_error())
    text = lib.tfrec_last_error().decode()
    for w in words:
        assert w in text, text


def quant(lib, X=A16, dt=0, n_rows=10, ldx=20, d=20, rows=None, n=10, q=A16, ldq=32, scale=A16):
    return lib.tfrec_quantize_rows_i8(None, X, dt, n_rows, ldx, d, rows, n, q, ldq, scale)


@pytest.mark.parametrize("kw,code,word", [
    (dict(), _lib.EINVAL, "null context"),
    (dict(dt=3), _lib.EINVAL, "type"),
    (dict(d=0), _lib.EINVAL, "shape"),
    (dict(n=-1), _lib.EINVAL, "shape"),
    (dict(ldx=19), _lib.EINVAL, "shape"),
    (dict(n=11), _lib.EINVAL, "rows"),
    (dict(rows=A16, n_rows=0), _lib.EINVAL, "rows"),
    (dict(rows=A16, n_rows=1 << 31), _lib.EINVAL, "rows"),
    (dict(X=None), _lib.EINVAL, "null"),
    (dict(scale=None), _lib.EINVAL, "null"),
    (dict(X=A16 + 2), _lib.EINVAL, "aligned"),
    (dict(X=A16 + 1, dt=1), _lib.EINVAL, "aligned"),
    (dict(X=A16 + 2, dt=1), _lib.EINVAL, "null context"),
    (dict(q=None), _lib.EINVAL, "null"),
    (dict(q=A16 + 8), _lib.EINVAL, "aligned"),
    (dict(ldq=16), _lib.EINVAL, "pitch"),
    (dict(ldq=40), _lib.EINVAL, "pitch"),
    (dict(n=0, n_rows=0, X=None, q=None, scale=None), _lib.EINVAL, "null context"),
])
def test_quantize_refusals(lib, kw, code, word):
    refused(lib, quant(lib, **kw), code, word)


def mm(lib, A=A16, lda=32, sa=A16, M=4, B=A16, ldb=32, sb=A16, N=5, K=20, bias=None, Cp=A16, dt=0, ldc=5):
    return lib.tfrec_matmul_i8(None, A, lda, sa, M, B, ldb, sb, N, K, bias, Cp, dt, ldc)


@pytest.mark.parametrize("kw,code,word", [
    (dict(), _lib.EINVAL, "null context"),
    (dict(dt=-1), _lib.EINVAL, "type"),
    (dict(K=0), _lib.EINVAL, "shape"),
    (dict(M=-1), _lib.EINVAL, "shape"),
    (dict(N=-1), _lib.EINVAL, "shape"),
    (dict(ldc=4), _lib.EINVAL, "shape"),
    (dict(K=131072, lda=131072, ldb=131072), _lib.EUNSUP, "131071"),
    (dict(lda=16), _lib.EINVAL, "pitch"),
    (dict(ldb=24), _lib.EINVAL, "pitch"),
    (dict(A=None), _lib.EINVAL, "A is null"),
    (dict(B=A16 + 4), _lib.EINVAL, "aligned"),
    (dict(sa=None), _lib.EINVAL, "null"),
    (dict(Cp=None), _lib.EINVAL, "null"),
    (dict(Cp=A16 + 2), _lib.EINVAL, "aligned"),
    (dict(Cp=A16 + 2, dt=2), _lib.EINVAL, "null context"),
])
def test_matmul_refusals(lib, kw, code, word):
    refused(lib, mm(lib, **kw), code, word)


def topk(lib, P=A16, ldp=32, sp=A16, U=9, compact=0, Q=A16, ldq=32, sq=A16, b=None, I=50, d=20, lo=0, hi=50, users=A16, n=3, tp=None, ti=None, k=5,
         ids=A16, sc=A16):
    return lib.tfrec_score_topk_i8(None, P, ldp, sp, U, compact, Q, ldq, sq, b, I, d, lo, hi, users, n, tp, ti, k, ids, sc)


@pytest.mark.parametrize("kw,code,word", [
    (dict(), _lib.EINVAL, "null context"),
    (dict(k=0), _lib.EINVAL, "shape"),
    (dict(n=-1), _lib.EINVAL, "shape"),
    (dict(d=0), _lib.EINVAL, "shape"),
    (dict(k=241), _lib.EUNSUP, "240"),
    (dict(d=257, ldp=272, ldq=272), _lib.EUNSUP, "256"),
    (dict(lo=3, hi=2), _lib.EINVAL, "range"),
    (dict(hi=51), _lib.EINVAL, "range"),
    (dict(lo=-1), _lib.EINVAL, "range"),
    (dict(I=1 << 31, hi=1 << 31), _lib.EUNSUP, "int32"),
    (dict(compact=2), _lib.EINVAL, "p_compact"),
    (dict(compact=1, U=2), _lib.EINVAL, "rows"),
    (dict(compact=1, U=3), _lib.EINVAL, "null context"),
    (dict(U=0, P=None), _lib.EINVAL, "rows"),
    (dict(tp=A16), _lib.EINVAL, "CSR"),
    (dict(ldp=16), _lib.EINVAL, "pitch"),
    (dict(Q=A16 + 8), _lib.EINVAL, "aligned"),
    (dict(users=None), _lib.EINVAL, "null"),
    (dict(sq=None), _lib.EINVAL, "null"),
    (dict(sq=None, lo=7, hi=7), _lib.EINVAL, "null context"),
])
def test_score_topk_refusals(lib, kw, code, word):
    refused(lib, topk(lib, **kw), code, word)


def clip(lib, grads, outs=None, counts=None, types=None, max_norm=1.0, n=None, norm=None):
    n = len(grads) if n is None else n
    counts = [4] * len(grads) if counts is None else counts
    types = [0] * len(grads) if types is None else types
    outs = grads if outs is None else outs
    m = max(1, len(grads))
    return lib.tfrec_grad_clip(None, n, (C.c_void_p * m)(*grads), (C.c_void_p * m)(*outs), (C.c_int64 * m)(*counts), (C.c_int * m)(*types), max_norm, norm)


G = [A16, A16 + 64, A16 + 128]


@pytest.mark.parametrize("kw,word", [
    (dict(grads=G), "null context"),
    (dict(grads=G, outs=[A16 + 512, A16 + 256, A16 + 768]), "null context"),
    (dict(grads=G, outs=[A16 + 256, A16 + 256 + 16, A16]), "does not replace"),        # the third writes the first gradient
    (dict(grads=G, outs=[A16 + 256, A16 + 264, A16 + 512]), "overlaps another output"),
    (dict(grads=G, outs=[A16 + 512, A16 + 512, A16 + 256]), "overlaps another output"),
    (dict(grads=[A16, A16]), "overlaps another output"),                               # the same tensor twice, in place
    (dict(grads=G, outs=[A16 + 4, A16 + 256, A16 + 512]), "does not replace"),         # shifted by one value
    (dict(grads=G, outs=[A16 + 64, A16 + 256, A16 + 512]), "does not replace"),
    (dict(grads=G, outs=[None, A16 + 256, A16 + 512]), "output 0 is null"),
    (dict(grads=G, outs=[A16 + 258, A16 + 512, A16 + 768]), "aligned"),
    (dict(grads=[None, A16], counts=[0, 4]), "null context"),                          # empty tensors need no buffer
    (dict(grads=[None, A16]), "tensor 0 is null"),
    (dict(grads=[A16 + 2]), "aligned"),
    (dict(grads=[A16 + 2], types=[1]), "null context"),
    (dict(grads=[A16], types=[3]), "type"),
    (dict(grads=[A16], counts=[-1]), "length"),
    (dict(grads=G, max_norm=0.0), "max_norm"),
    (dict(grads=G, max_norm=-1.0), "max_norm"),
    (dict(grads=G, max_norm=float("inf")), "max_norm"),
    (dict(grads=G, max_norm=float("nan")), "max_norm"),
    (dict(grads=G, n=-1), "tensors"),
    (dict(grads=G, norm=A16 + 1), "misaligned"),
    (dict(grads=[]), "null context"),
])
def test_clip_refusals(lib, kw, word):
    refused(lib, clip(lib, **kw), _lib.EINVAL, word)


def test_overlap_check_on_many_random_ranges(lib):
    """Against the plain quadratic rule: outputs disjoint, and none over a gradient but its own."""
    rng = np.random.default_rng(3)
    verdicts = set()
    for _ in range(300):
        n = int(rng.integers(1, 12))
        counts = rng.integers(0, 9, n)
        g = A16 + 4 * rng.integers(0, 400, n)
        inplace = rng.random(n) < 0.5
        o = np.where(inplace, g, A16 + 4 * rng.integers(0, 400, n))
        ok = True
        for i in range(n):
            for j in range(n):
                if counts[i] == 0 or counts[j] == 0:
                    continue
                over = lambda a, b: a < b + 4 * counts[j] and b < a + 4 * counts[i]      # noqa: E731
                if i != j and over(o[i], o[j]):
                    ok = False
                if over(o[i], g[j]) and not (i == j and o[i] == g[j]):
                    ok = False
        rc = clip(lib, [int(x) for x in g], [int(x) for x in o], [int(c) for c in counts])
        assert rc == _lib.EINVAL
        assert (b"null context" in lib.tfrec_last_error()) == ok
        verdicts.add(ok)
    assert verdicts == {True, False}


def test_norm_refusals(lib):
    one = (C.c_void_p * 1)(A16), (C.c_int64 * 1)(4), (C.c_int * 1)(0)
    refused(lib, lib.tfrec_grad_norm(None, 1, *one, None), _lib.EINVAL, "output")
    refused(lib, lib.tfrec_grad_norm(None, 1, None, None, None, A16), _lib.EINVAL, "host array")
    refused(lib, lib.tfrec_grad_norm(None, 1, *one, A16), _lib.EINVAL, "null context")


class _Host:
    """A stand-in with a shape and a dtype, and no device memory behind it."""

    def __init__(self, *shape, dtype="int8"):
        self.shape, self.dtype = shape, np.dtype(dtype)


def test_python_refusals():
    import torch
    from tfrec_amd.device import GradList, QuantRows
    with pytest.raises(ValueError, match="int8"):
        QuantRows(_Host(4, 32, dtype="uint8"), _Host(4, dtype="float32"), 20)
    with pytest.raises(ValueError, match="scale"):
        QuantRows(_Host(4, 32), _Host(5, dtype="float32"), 20)
    with pytest.raises(ValueError, match="multiple of 16"):
        QuantRows(_Host(4, 24), _Host(4, dtype="float32"), 20)
    with pytest.raises(ValueError, match="multiple of 16"):
        QuantRows(_Host(4, 16), _Host(4, dtype="float32"), 20)
    with pytest.raises(ValueError, match="contiguous"):
        QuantRows(torch.zeros(4, 64, dtype=torch.int8)[:, :32], torch.zeros(4), 20)

    class Dev:
        device = 0
    with pytest.raises(ValueError, match="is on cpu"):
        GradList(Dev(), [torch.zeros(3)])
    with pytest.raises(ValueError, match="float64"):
        GradList(Dev(), [torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="1 outputs for 2"):
        GradList(Dev(), [torch.zeros(3), torch.zeros(3)], out=[torch.zeros(3)])


def test_configuration_refusals():
    from tfrec_amd.model.APR import APR
    from tfrec_amd.model.BPR import clip_norm_of
    assert clip_norm_of({}) == 0.0 and clip_norm_of({"clip_norm": 2}) == 2.0
    for bad in (-1.0, float("nan"), float("inf"), "1.0", None, True):
        with pytest.raises(ValueError, match="clip_norm"):
            clip_norm_of({"clip_norm": bad})
    with pytest.raises(ValueError, match="BPR and DNSBPR"):
        APR(None, {"clip_norm": 1.0}, None, None)
    import scipy.sparse as sp
    from tfrec_amd.evaluator import FoldOutEvaluator
    m = sp.csr_matrix(np.eye(3, dtype=np.float32))
    assert FoldOutEvaluator.from_config({"score_dtype": "i8"}, m, m).score_mode == _lib.SCORE_I8
    with pytest.raises(ValueError, match="score_dtype"):
        FoldOutEvaluator(m, m, score_dtype="i4")


def test_list_refusals(lib):
    h = C.c_void_p()
    one = (C.c_void_p * 1)(A16), (C.c_void_p * 1)(A16 + 4), (C.c_int64 * 1)(4), (C.c_int * 1)(0)
    refused(lib, lib.tfrec_grads_create(None, 1, *one, C.byref(h)), _lib.EINVAL, "does not replace")
    refused(lib, lib.tfrec_grads_create(None, 1, one[0], one[0], one[2], one[3], None), _lib.EINVAL, "out is null")
    refused(lib, lib.tfrec_grads_create(None, 1, one[0], one[0], one[2], one[3], C.byref(h)), _lib.EINVAL, "null context")
    assert h.value is None
    refused(lib, lib.tfrec_grads_norm(None, None, A16), _lib.EINVAL, "null list")
    refused(lib, lib.tfrec_grads_clip(None, None, 1.0, A16), _lib.EINVAL, "null list")
    assert lib.tfrec_grads_destroy(None, None) == _lib.OK


def test_gradient_tables_that_overlap_are_refused(lib):
    U, I, d = 10, 20, 8
    P, Q, b, gP, gQ, gb = (A16 + k * 4096 for k in range(6))

    def call(**kw):
        t = dict(P=P, Q=Q, b=b, gP=gP, gQ=gQ, gb=gb)
        t.update(kw)
        return lib.tfrec_bpr_grads(None, t["P"], t["Q"], t["b"], U, I, d, A16, A16, A16, 5, 0.1, t["gP"], t["gQ"], t["gb"], None)
    refused(lib, call(), _lib.EINVAL, "null context")
    refused(lib, call(gP=None), _lib.EINVAL, "null gradient")
    for kw in (dict(gQ=gP), dict(gb=gQ + I * d * 4 - 4), dict(gP=gQ - U * d * 4 + 4), dict(gb=gP)):
        refused(lib, call(**kw), _lib.EINVAL, "two gradient tables overlap")
    for kw in (dict(gP=P), dict(gQ=Q + 4), dict(gb=b), dict(gP=Q), dict(gb=P + U * d * 4 - 4)):
        refused(lib, call(**kw), _lib.EINVAL, "overlaps the parameters")
    refused(lib, call(gQ=gP + U * d * 4, gb=gP + (U + I) * d * 4), _lib.EINVAL, "null context")
