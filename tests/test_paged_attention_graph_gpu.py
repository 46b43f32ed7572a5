"""paged_attention in captured graphs: without an eager call before, at sizes past the warm-up's, and with the
parts joined by a second kernel.  Every replay is checked, with eager work between them."""
import pytest
import torch

from test_paged_attention_gpu import check, make
from test_paged_attention_threads_gpu import two_calls

pytestmark = pytest.mark.gpu


def capture(stream, args, **kw):
    from powershard_amd import ops
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = ops.paged_attention(*args, **kw)
    return graph, out


def shift(args):
    """New queries in place."""
    args[0].copy_(args[0].roll(1, 0).roll(3, 2))


def test_two_graphs_without_a_warm_up(gpu):
    """The second one captured is replayed first: nothing of it may be left to the first."""
    from powershard_amd import ops
    stream = torch.cuda.Stream(gpu)
    calls = [make([2000, 777], 40, 8, 128, 16, "int8", torch.bfloat16, gpu, seed=s) for s in (1, 2)]
    torch.cuda.synchronize()
    graphs = [capture(stream, args) for args in calls]
    for i in (1, 0, 1, 1, 0):
        graph, out = graphs[i]
        shift(calls[i])
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, calls[i])
        with torch.cuda.stream(stream):
            eager = ops.paged_attention(*calls[1 - i])
        stream.synchronize()
        check(eager, calls[1 - i])


def test_a_call_larger_than_the_warm_up(gpu):
    from powershard_amd import ops
    stream = torch.cuda.Stream(gpu)
    small = make([300], 8, 8, 64, 16, "int8", torch.bfloat16, gpu, seed=3)
    large = make([4000, 3000, 2500, 100, 4000, 1], 40, 8, 128, 16, "int8", torch.bfloat16, gpu, seed=4)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ops.paged_attention(*small)
    stream.synchronize()
    graph, out = capture(stream, large)
    for _ in range(4):
        with torch.cuda.stream(stream):       # (its workspace grows here)
            eager = ops.paged_attention(*large)
        stream.synchronize()
        check(eager, large)
        shift(large)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, large)


@pytest.mark.parametrize("which", [0, 1])
def test_parts_joined_by_a_second_kernel(gpu, which):
    """The bits of the eager call, whose parts are elsewhere."""
    from powershard_amd import ops
    stream = torch.cuda.Stream(gpu)
    args = two_calls(gpu)[which]
    other = two_calls(gpu)[1 - which]
    torch.cuda.synchronize()
    graph, out = capture(stream, args)
    for _ in range(4):
        shift(args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        ops.paged_attention(*other)
        assert torch.equal(got, ops.paged_attention(*args))
    check(got, args)
