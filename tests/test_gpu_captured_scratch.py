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


# ------------------------------------------------------------------------------------------------------------- training
def problem(U, I, d, B, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tables = [torch.randn(s, generator=g, device="cuda") * 0.1 for s in ((U, d), (I, d), (I,))]
    batch = [torch.randint(0, n, (B,), generator=g, device="cuda", dtype=torch.int32) for n in (U, I, I)]
    return g, tables, batch, [torch.full_like(t, 7.0) for t in tables]


def test_a_captured_clipped_step(ctx):
    """Gradients, clipping and the three axpys in one graph, replayed on new batches; between the replays eager steps on a much
    larger batch, for which the workspace has grown."""
    dev, stream = ctx
    U, I, d, B = 30000, 20000, 64, 50000
    g, tables, batch, grads = problem(U, I, d, B, 1)
    _, tables2, big, grads2 = problem(U, I, d, 40 * B, 2)
    lst, norm, loss = dev.grad_list(grads), torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    mine = [t.clone() for t in tables]

    def step(to):
        dev.bpr_grads(*to, *batch, 0.01, *grads, loss=loss)
        dev.clip_grads(lst, 0.5, norm=norm)
        for t, x in zip(to, grads):
            dev.axpy(t, x, -0.05, n=t.numel())
    _, narrow, _, to_narrow = problem(U, I, 4, 1, 9)
    dev.bpr_grads(*narrow, *big, 0.01, *to_narrow)            # (room for the larger batch's index, and for short rows)
    step([t.clone() for t in tables])
    graph = capture(stream, lambda: step(tables))
    old = dev.workspace_bytes()
    taken = memory_taken(lambda: dev.bpr_grads(*tables2, *big, 0.01, *grads2))
    assert 2 * MARGIN < old < dev.workspace_bytes() and taken >= dev.workspace_bytes() - MARGIN, "the block that the graph names was given back"
    for turn in range(3):
        for x in batch:
            x.copy_(x[torch.randperm(B, generator=g, device="cuda")])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in tables + grads + [norm, loss]]
        step(mine)
        torch.cuda.synchronize()
        for a, b in zip(got, mine + grads + [norm, loss]):
            assert torch.equal(a, b)
        assert float(norm) > 0.5
        dev.bpr_grads(*tables2, *big, 0.01, *grads2)
        dev.synchronize()


def test_the_index_of_a_captured_batch_is_kept(ctx):
    """The sorted index lies outside the workspace: a larger batch replaces its block, and frees it only where no graph names it."""
    from tfrec_amd.device import Device
    dev, stream = ctx
    U, I, d, B = 30000, 20000, 4, 600000
    _, tables, batch, grads = problem(U, I, d, B, 3)
    _, _, big, grads2 = problem(U, I, d, 3 * B, 4)
    fresh = Device(0, stream.cuda_stream)
    for c in (fresh, dev):
        c.reserve(max_batch=3 * B, d=d)

    def step(c, to=grads):
        c.bpr_grads(*tables, *batch, 0.01, *to)
    ws = dev.workspace_bytes()
    step(fresh)
    big_after_small = memory_taken(lambda: fresh.bpr_grads(*tables, *big, 0.01, *grads2))        # (frees the smaller block)
    small = memory_taken(lambda: step(dev))
    assert dev.workspace_bytes() == ws and fresh.workspace_bytes() == ws and small >= MARGIN
    graph = capture(stream, lambda: step(dev))
    taken = memory_taken(lambda: dev.bpr_grads(*tables, *big, 0.01, *grads2))
    assert taken >= big_after_small + small / 2, "the index block that the graph names was given back"
    other = torch.full((small,), 0x5a, dtype=torch.uint8, device="cuda")
    want = [torch.empty_like(x) for x in grads]
    for turn in range(3):
        for x in batch:
            x.copy_(x.flip(0) if turn else x.roll(1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(fresh, want)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want)) and bool((other == 0x5a).all())
        for x in grads:
            x.fill_(3.0)
        dev.bpr_grads(*tables, *big, 0.01, *grads2)
    torch.cuda.synchronize()
    fresh.close()


def test_gradients_that_lack_scratch_are_refused_under_capture(ctx):
    """First for the workspace, then, with that reserved, for the index; neither call records a launch."""
    dev, stream = ctx
    _, tables, batch, grads = problem(300, 200, 8, 5000, 5)
    x = torch.zeros(4, device="cuda")

    def step():
        with pytest.raises(MemoryError, match="captured"):
            dev.bpr_grads(*tables, *batch, 0.01, *grads)
        x.add_(1.0)
    for turn in range(2):
        graph = capture(stream, step)
        graph.replay()
        torch.cuda.synchronize()
        assert (x == turn + 1.0).all() and all(bool((t == 7.0).all()) for t in grads)
        dev.reserve(max_batch=5000, d=8)
    dev.bpr_grads(*tables, *batch, 0.01, *grads)
    dev.synchronize()
    assert not bool((grads[0] == 7.0).any())
