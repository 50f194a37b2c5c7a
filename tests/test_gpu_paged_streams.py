"""A workspace that PagedAttention allocates itself, on streams other than the one that it was allocated on."""
import pytest

pytestmark = pytest.mark.gpu


def _call(q, **more):
    """(cache, tensors that PagedAttention takes) of a small call."""
    import torch
    import pitch_amd as P
    dev, d, kv, page = q.device, 64, 2, 16
    cfg = q.config("turboQuant", d, 4)
    cache = P.PagedCache(q, cfg, cfg, pages=80, pageSize=page, kvHeads=kv)
    x = torch.randn(80 * page, kv, d, device=dev).to(torch.bfloat16)
    cache.enqueueAppend(x, x.flip(0).contiguous(), torch.arange(80 * page, device=dev))
    queries = torch.randn(1, 4, d, device=dev).to(torch.bfloat16)
    args = (queries, torch.arange(80, dtype=torch.int32, device=dev)[None], torch.tensor([80 * page], dtype=torch.int32, device=dev))
    return cache, args


def _busy(stream, ms=30):
    """Work of about this long (a kernel that counts clocks and ends)."""
    import torch
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 1e6))


@pytest.mark.parametrize("form", ["stream", "handle", "current stream"])
def test_work_that_still_uses_the_memory_comes_first(q, form):
    """The memory may be a block whose last user still runs on the stream of the allocation."""
    import torch
    import pitch_amd as P
    cache, args = _call(q)
    out, ref = torch.zeros_like(args[0]), torch.zeros_like(args[0])
    cache.enqueueAttention(*args, ref)
    other, main = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    _busy(main)
    done = main.record_event()
    step = P.PagedAttention(cache, *args, out)
    if form == "current stream":
        with torch.cuda.stream(other):
            step.enqueue()
    else:
        step.enqueue(other if form == "stream" else other.cuda_stream)
    assert not done.query(), "the main stream's work has ended early: nothing is tested"
    other.synchronize()
    assert done.query()
    assert torch.equal(out, ref)


def test_the_memory_is_kept_while_a_stream_uses_it(q):
    """Dropped while another stream still has the call ahead, the workspace does not go to the next allocation."""
    import torch
    import pitch_amd as P
    cache, args = _call(q)
    out, ref = torch.zeros_like(args[0]), torch.zeros_like(args[0])
    cache.enqueueAttention(*args, ref)
    nbytes = cache.attentionWorkspaceBytes(1, 2)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    step = P.PagedAttention(cache, *args, out)
    step.enqueue(other)
    other.synchronize()
    _busy(other)
    step.enqueue(other)
    used = step._call.workspace
    del step
    new = [torch.empty(nbytes, dtype=torch.uint8, device=q.device) for _ in range(3)]
    taken = used in [t.data_ptr() for t in new]
    assert not other.query(), "the other stream's work has ended early: nothing is tested"
    assert not taken, "the workspace was handed out while a call ahead uses it"
    other.synchronize()
    assert torch.equal(out, ref)


def test_a_graph_of_a_call_with_a_workspace_of_its_own(q):
    """Captured on a side stream, replayed on two streams in turn, eager calls on others in between."""
    import torch
    import pitch_amd as P
    cache, args = _call(q)
    out, ref = torch.zeros_like(args[0]), torch.zeros_like(args[0])
    step = P.PagedAttention(cache, *args, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step.enqueue()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        args[0].copy_(torch.randn(args[0].shape).to(torch.bfloat16))
        out.zero_()
        cache.enqueueAttention(*args, ref)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i % 2]):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        step.enqueue(streams[(i + 1) % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
