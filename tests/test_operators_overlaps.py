"""Outputs that overlap what a call still reads or writes are refused, not raced: the checks are the host's, so all of this runs
without a GPU (see test_operators_refusals.py)."""
import ctypes as C

import numpy as np
import pytest

from tfrec_amd import _lib

A = 1 << 20              # an address that is aligned and never read


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, rc, *words):
    assert rc == _lib.EINVAL, (rc, lib.tfrec_last_error())
    text = lib.tfrec_last_error().decode()
    for w in words:
        assert w in text, text


def clip(lib, grads, outs, counts, types, norm):
    n = len(grads)
    return lib.tfrec_grad_clip(None, n, (C.c_void_p * n)(*grads), (C.c_void_p * n)(*outs), (C.c_int64 * n)(*counts), (C.c_int * n)(*types), 1.0, norm)


def test_a_norm_within_a_tensor_is_refused(lib):
    grads, outs, counts, types = [A, A + 4096, A + 8192], [A, A + 65536, A + 8192], [100, 33, 0], [0, 1, 0]
    for norm, word in ((A, "tensor 0"), (A + 396, "tensor 0"), (A + 400, "null context"), (A - 4, "null context"), (A + 4096, "tensor 1"), (A + 4096 + 64, "tensor 1"),
                       (A + 4096 + 68, "null context"), (A + 65536, "tensor 1"), (A + 65536 + 64, "tensor 1"), (A + 65536 + 68, "null context"),
                       (A + 8192, "null context"), (None, "null context")):                       # (the third tensor is empty)
        refused(lib, clip(lib, grads, outs, counts, types, norm), word)


def bytes_of(at, pitch, length, n):
    return {at + r * pitch + i for r in range(n) for i in range(length)}


def test_rows_overlap_against_sets_of_bytes(lib):
    f = lib.tfrec_rows_overlap
    f.argtypes, f.restype = [C.c_size_t] + [C.c_int64] * 3 + [C.c_size_t] + [C.c_int64] * 3, C.c_int
    rng = np.random.default_rng(1)
    verdicts = [0, 0]
    for _ in range(4000):
        rows = []
        for _ in range(2):
            length, n = int(rng.integers(0, 12)), int(rng.integers(0, 7))
            rows.append((1000 + int(rng.integers(0, 80)), length + int(rng.integers(0, 20)) or 1, length, n))
        if rng.random() < 0.3:                        # columns of one matrix
            rows[1] = (rows[1][0], rows[0][1], min(rows[1][2], rows[0][1]), rows[1][3])
        want = bool(bytes_of(*rows[0]) & bytes_of(*rows[1]))
        assert f(*rows[0], *rows[1]) == want == f(*rows[1], *rows[0]), rows
        verdicts[want] += 1
    assert min(verdicts) > 500


def test_rows_overlap_far_out(lib):
    """Spans beyond 2^32 bytes, a vector between a matrix's rows, and one that crosses from a gap into a row."""
    f = lib.tfrec_rows_overlap
    f.argtypes, f.restype = [C.c_size_t] + [C.c_int64] * 3 + [C.c_size_t] + [C.c_int64] * 3, C.c_int
    at, pitch, length, n = 1 << 40, 1 << 20, 1000, 1 << 16
    row = at + 60000 * pitch
    for lo, size, want in ((row, 4, 1), (row + 999, 4, 1), (row + 1000, pitch - 1000, 0), (row + 1000, pitch - 999, 1), (row - 4, 4, 0), (row - 4, 5, 1),
                           (at + n * pitch, 4, 0), (at + (n - 1) * pitch + 1000, 4, 0), (at - 4, 4, 0), (at - 4, 5, 1), (at - 4, 1 << 40, 1)):
        assert f(at, pitch, length, n, lo, size, size, 1) == want == f(lo, size, size, 1, at, pitch, length, n), (lo, size)


def test_gradients_whose_indices_or_loss_lie_in_a_table_are_refused(lib):
    U, I, d, B = 10, 20, 8, 50
    tables = {k: A + i * 4096 for i, k in enumerate(("P", "Q", "b", "gP", "gQ", "gb"))}
    lists = {k: A + 65536 + i * 4096 for i, k in enumerate(("users", "pos", "neg"))}

    def call(loss=None, B=B, **kw):
        t = dict(tables, **lists)
        t.update(kw)
        return lib.tfrec_bpr_grads(None, t["P"], t["Q"], t["b"], U, I, d, t["users"], t["pos"], t["neg"], B, 0.1, t["gP"], t["gQ"], t["gb"], loss)
    refused(lib, call(), "null context")
    refused(lib, call(loss=A + 131072), "null context")
    for k in lists:
        for g, size in (("gP", U * d * 4), ("gQ", I * d * 4), ("gb", I * 4)):
            refused(lib, call(**{k: tables[g] + size - 4}), "overlaps")
            refused(lib, call(**{k: tables[g] - B * 4 + 4}), "overlaps")
            refused(lib, call(**{k: tables[g] + size}), "null context")
            refused(lib, call(B=0, **{k: tables[g]}), "null context")
        refused(lib, call(**{k: tables["Q"]}), "null context")               # (two inputs)
    for k, at in list(tables.items()) + list(lists.items()):
        refused(lib, call(loss=at), "loss")
        refused(lib, call(loss=at - 8), "loss")
        refused(lib, call(loss=at - 16), "null context")


class _Buffer:
    """A shape, a type and a GPU, and no memory."""

    def __init__(self, *shape, dtype="float32", gpu=0):
        self.shape, self.dtype, self.gpu = shape, np.dtype(dtype), gpu

    def get_device(self):
        return self.gpu

    def data_ptr(self):
        raise AssertionError("an address was asked for")


def test_gradient_buffers_of_another_type_size_or_place_are_refused():
    """Their kernels write whole tables: a narrower type or a shorter table would be written past its end."""
    from tfrec_amd.device import Device

    class Dev:
        device, lib, h = 0, None, None
    U, I, d, B = 4, 5, 8, 3

    def call(loss=None, **kw):
        t = dict(P=_Buffer(U, d), Q=_Buffer(I, d), b=_Buffer(I), users=_Buffer(B, dtype="int32"), pos=_Buffer(B, dtype="int32"), neg=_Buffer(B, dtype="int32"),
                 gP=_Buffer(U, d), gQ=_Buffer(I, d), gb=_Buffer(I))
        t.update(kw)
        return Device.bpr_grads(Dev(), t["P"], t["Q"], t["b"], t["users"], t["pos"], t["neg"], 0.1, t["gP"], t["gQ"], t["gb"], loss=loss)
    with pytest.raises(AttributeError):             # (in order: the library is asked for, and there is none)
        call(loss=_Buffer(2, dtype="float64"))
    for name, shape in (("P", (U, d)), ("Q", (I, d)), ("b", (I,)), ("gP", (U, d)), ("gQ", (I, d)), ("gb", (I,))):
        for bad in (_Buffer(*shape, dtype="float16"), _Buffer(*shape, dtype="float64"), _Buffer(*shape, gpu=1), _Buffer(*shape, gpu=-1), np.zeros(shape, np.float32)):
            with pytest.raises(ValueError, match="float32"):
                call(**{name: bad})
    for name in ("users", "pos", "neg"):
        with pytest.raises(ValueError, match="int32"):
            call(**{name: _Buffer(B, dtype="int64")})
        with pytest.raises(ValueError, match="int32"):
            call(**{name: _Buffer(B, dtype="int32", gpu=2)})
    for kw in (dict(Q=_Buffer(I, d + 1)), dict(b=_Buffer(I - 1)), dict(pos=_Buffer(B - 1, dtype="int32")), dict(neg=_Buffer(B - 1, dtype="int32")),
               dict(gP=_Buffer(U - 1, d)), dict(gb=_Buffer(I - 1)), dict(loss=_Buffer(1, dtype="float64"))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError, match="float64"):
        call(loss=_Buffer(2))
