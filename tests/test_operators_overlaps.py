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
