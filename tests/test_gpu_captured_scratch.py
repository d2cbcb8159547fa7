"""Scratch that a captured HIP graph names: the context keeps it when a later call needs more, so a replay reads and writes
memory that is still its own.  Every test looks at the card's free memory first and replays only once it has seen that the old
block was kept."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture()
def ctx():
    """A context of its own (its workspace is empty) on a stream of its own."""
    from tfrec_amd.device import Device
    stream = torch.cuda.Stream()
    dev = Device(0, stream.cuda_stream)
    with torch.cuda.stream(stream):
        yield dev, stream
    torch.cuda.synchronize()
    dev.close()


def capture(stream, f):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        f()
    torch.cuda.synchronize()
    return graph


def memory_taken(f):
    """Bytes of the card's memory that f took and did not give back."""
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    f()
    torch.cuda.synchronize()
    return before - torch.cuda.mem_get_info()[0]


MARGIN = 8 << 20        # (allocations are rounded up)


def outgrow(dev, rows=200000):
    """Makes the workspace grow; -> (its size before, what growing took from the card)."""
    R = torch.zeros(rows, 8, device="cuda")
    ids, sc = torch.zeros(rows, 2, dtype=torch.int32, device="cuda"), torch.zeros(rows, 2, device="cuda")
    old = dev.workspace_bytes()
    taken = memory_taken(lambda: dev.topk_dense(R, 2, out_ids=ids, out_scores=sc))
    assert dev.workspace_bytes() > old + 4 * MARGIN
    return old, taken


def lists(n, k):
    return torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")


@pytest.mark.parametrize("I", [2000, 5000])
def test_quantised_tables_of_a_captured_score_mode(ctx, I):
    """score_topk in the 8-bit mode holds both tables in the workspace, on either side of the 4096 items up to which nothing else
    of the call does."""
    from tfrec_amd.device import SCORE_I8
    dev, stream = ctx
    g = torch.Generator(device="cuda").manual_seed(I)
    n, d, k = 200000, 256, 3
    P, Q, b = torch.randn(n, d, generator=g, device="cuda"), torch.randn(I, d, generator=g, device="cuda"), torch.randn(I, generator=g, device="cuda")
    users = torch.arange(n, dtype=torch.int32, device="cuda")
    ids, sc = lists(n, k)

    def step():
        dev.score_topk(P, Q, b, users, k, mode=SCORE_I8, out_ids=ids, out_scores=sc)
    step()
    graph = capture(stream, step)
    old, taken = outgrow(dev)
    assert old > 4 * MARGIN and taken >= dev.workspace_bytes() - MARGIN, "the block that the graph names was given back"
    other = torch.full((old,), 0x5a, dtype=torch.uint8, device="cuda")        # would lie in it, had it been
    for turn in range(3):
        Q.copy_(torch.randn(I, d, generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = ids.clone(), sc.clone()
        ids.zero_(), sc.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], ids) and torch.equal(got[1], sc)
        assert bool((other == 0x5a).all())


def test_bounds_of_a_captured_topk(ctx):
    """Kept tables and more than 4096 items: the workspace holds the bounds of the first step."""
    dev, stream = ctx
    g = torch.Generator(device="cuda").manual_seed(3)
    n, I, d, k = 5000, 50000, 32, 10
    p, q = dev.quantize_rows(torch.randn(n, d, generator=g, device="cuda")), dev.quantize_rows(torch.randn(I, d, generator=g, device="cuda"))
    users = torch.arange(n, dtype=torch.int32, device="cuda")
    ids, sc = lists(n, k)

    def step():
        dev.score_topk_i8(p, q, None, users, k, out_ids=ids, out_scores=sc)
    step()
    graph = capture(stream, step)
    old, taken = outgrow(dev)
    assert old > 4 * MARGIN and taken >= dev.workspace_bytes() - MARGIN, "the block that the graph names was given back"
    other = torch.full((old,), 0x5a, dtype=torch.uint8, device="cuda")
    for turn in range(3):
        dev.quantize_rows(torch.randn(n, d, generator=g, device="cuda"), out=p)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = ids.clone(), sc.clone()
        ids.zero_(), sc.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], ids) and torch.equal(got[1], sc)
        assert bool((other == 0x5a).all())


def test_a_workspace_that_no_graph_names_is_given_back(ctx):
    dev, _ = ctx
    outgrow(dev, 60000)
    old, taken = outgrow(dev)
    assert old > 4 * MARGIN and taken <= dev.workspace_bytes() - old + MARGIN


def test_the_workspace_does_not_grow_under_capture(ctx):
    """A captured call that needs more than there is is refused; the capture, and the calls behind it, are not spoilt."""
    from tfrec_amd.device import SCORE_I8
    dev, stream = ctx
    P, Q, b = torch.randn(300, 16, device="cuda"), torch.randn(500, 16, device="cuda"), torch.zeros(500, device="cuda")
    users, x = torch.arange(300, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    ids, sc = lists(300, 5)

    def step():
        with pytest.raises(MemoryError, match="captured"):
            dev.score_topk(P, Q, b, users, 5, mode=SCORE_I8, out_ids=ids, out_scores=sc)
        x.add_(1.0)
    graph = capture(stream, step)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert (x == 3.0).all() and not ids.any()
    dev.score_topk(P, Q, b, users, 5, mode=SCORE_I8, out_ids=ids, out_scores=sc)
    dev.synchronize()
    assert ids.any()
