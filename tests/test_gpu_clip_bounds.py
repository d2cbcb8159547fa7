"""Gradient clipping where the bound is no float32, and where the factor leaves float32's range: the factor and the product are
formed in 64 bits, so that a scaled value is one rounding (two for 16-bit types) off."""
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


HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}            # half a step of the type the product is rounded to next
TINY = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}          # the same among its subnormal numbers


def clip_all_ways(dev, host, bound):
    """The scaled tensors in place, out of place and through a kept list."""
    for kind in ("in place", "out of place", "kept list"):
        grads = [x.cuda() for x in host]
        out = [torch.full_like(x, 5.0) for x in grads] if kind == "out of place" else grads
        norm = torch.zeros(1, device="cuda")
        if kind == "kept list":
            dev.clip_grads(dev.grad_list(grads), bound, norm=norm)
        else:
            dev.clip_grads(grads, bound, out=out if out is not grads else None, norm=norm)
        dev.synchronize()
        yield kind, [x.cpu() for x in out], float(norm)


def check(dev, host, bound):
    total = sum(float(np.sum(np.square(x.double().numpy()))) for x in host)
    norm = np.sqrt(total)
    s = bound / max(norm, bound)
    for kind, got, n in clip_all_ways(dev, host, bound):
        if norm < 3.4e38:
            assert abs(n - norm) <= 2.0 ** -23 * norm
        for x, y in zip(host, got):
            want = x.double() * s
            # half a step of float32 (and of the type), a millionth more for the order of the norm's sum; half a subnormal step
            tol = want.abs() * ((2.0 ** -24 + HALF[x.dtype] * (1 + 2.0 ** -24)) * (1 + 1e-6)) + (2.0 ** -150 + TINY[x.dtype]) * (1 + 1e-6)
            off = (y.double() - want).abs()
            assert (off <= tol).all(), (kind, x.dtype, float((off / tol).max()), bound)


@pytest.mark.parametrize("lengths", [[1], [300, 7], [40000, 5000, 3], [9000] * 3 + [200001], [701] * 130], ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_bounds_that_are_no_float32(dev, lengths):
    g = torch.Generator().manual_seed(sum(lengths))
    host = [(torch.randn(n, generator=g) * 0.1).to((torch.float32, torch.bfloat16, torch.float32, torch.float16)[i % 4]) for i, n in enumerate(lengths)]
    norm = float(np.sqrt(sum(float(np.sum(np.square(x.double().numpy()))) for x in host)))
    for part in (0.1, 0.3, 1 / 3, 0.7, 0.9, 0.99999999):
        check(dev, host, part * norm)


@pytest.mark.parametrize("n", [5, 100000])
@pytest.mark.parametrize("size,bound", [(1e30, 1e-38), (1e30, 3e-39), (3e38, 1e-40), (3e38, 1.0), (1e37, 1e-30), (1e25, 2e-36), (1e-30, 1e-42), (1e-10, 1e-44)])
def test_factors_beyond_the_range_of_float32(dev, n, size, bound):
    g = torch.Generator().manual_seed(n)
    x = (torch.rand(n, generator=g, dtype=torch.float64) * 2 - 1) * size
    x[::3] *= 1e-5
    check(dev, [x.float()], bound)


def test_bounds_beyond_the_range_of_float32(dev):
    """A bound above every float32 leaves all as it is, one below every float32 leaves zeros."""
    x = torch.randn(20000, generator=torch.Generator().manual_seed(1))
    for _, got, n in clip_all_ways(dev, [x], 1e300):
        assert torch.equal(got[0], x)
    for _, got, n in clip_all_ways(dev, [x], 1e-60):
        assert not got[0].any()


def test_a_norm_within_a_kept_tensor_is_refused(dev):
    """The norm of a list may lie anywhere but in a gradient or an output of it."""
    flat, to = torch.ones(3000, device="cuda"), torch.ones(3000, device="cuda")
    for out in (None, [to[0:500], to[800:900], to[1000:2000]]):
        lst = dev.grad_list([flat[0:500], flat[400:500], flat[1000:2000]] if out else [flat[0:500], flat[500:600], flat[1000:2000]], out=out)
        inside = [flat[0:1], flat[499:500], flat[1000:1001], flat[1999:2000]] + ([to[0:1], to[800:801], to[1999:2000]] if out else [flat[599:600]])
        for norm in inside:
            before = flat.clone(), to.clone()
            with pytest.raises(ValueError, match="norm"):
                dev.clip_grads(lst, 1.0, norm=norm)
            dev.synchronize()
            assert torch.equal(before[0], flat) and torch.equal(before[1], to)
        outside = [flat[700:701], flat[999:1000], flat[2000:2001], to[500:501] if out else to[0:1]]
        for norm in outside:
            dev.clip_grads(lst, 1e6, norm=norm)
            dev.synchronize()
            assert float(norm) > 1.0
            norm.fill_(1.0)
