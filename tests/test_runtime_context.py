"""Scratch and streams of the contexts that the Python calls use. No GPU: host scratch stands for device scratch, and stream
handles are numbers that nothing looks into."""
import ctypes
import queue
import threading
from ctypes import byref, c_int64, c_void_p

import pytest
import torch

HOST = 0   # diopi_host


@pytest.fixture()
def rt(built_libs):
    rt = built_libs.rt
    rt.diopiRequireBuffer.argtypes = [c_void_p, ctypes.POINTER(c_void_p), c_int64, ctypes.c_int]
    rt.diopiGetTensorData.argtypes = [c_void_p, ctypes.POINTER(c_void_p)]
    return rt


@pytest.fixture()
def ctx(rt):
    from diopi_b200.runtime import Context
    c = Context(None)
    yield c
    c.set_stream(0)   # no made-up stream is left when the context goes


def scratch(rt, ctx, nbytes=1000):
    t, p = c_void_p(), c_void_p()
    assert rt.diopiRequireBuffer(ctx.handle, byref(t), nbytes, HOST) == 0
    assert rt.diopiGetTensorData(t, byref(p)) == 0
    return p.value


def test_scratch_of_one_stream_is_not_handed_to_another(rt, ctx):
    """What a stream's kernels may still be using when its scratch is released is not ready for another stream's."""
    ctx.set_stream(0x100)
    a = scratch(rt, ctx)
    ctx.release()
    ctx.set_stream(0x200)
    b = scratch(rt, ctx)
    assert a != b
    ctx.release()
    ctx.set_stream(0x100)
    assert scratch(rt, ctx, 900) == a
    assert scratch(rt, ctx, 900) not in (a, b)
    ctx.release()
    ctx.set_stream(0x200)
    assert scratch(rt, ctx) == b
    assert ctx.stats()["blocks"] == 3


def test_scratch_of_a_stream_is_used_again(rt, ctx):
    first = scratch(rt, ctx)
    for _ in range(5):
        ctx.release()
        ctx.set_stream(0)
        assert scratch(rt, ctx) == first
    assert ctx.stats()["blocks"] == 1


def test_each_thread_has_a_default_context(built_libs):
    """A call sets the stream and then launches: between the two no other thread may set another one."""
    from diopi_b200.runtime import default_context
    mine, others, together = default_context(), [], threading.Barrier(3)

    def work():
        together.wait()      # all three alive at once: an identifier of a thread that has ended may come again
        others.append(default_context())
        together.wait()

    ts = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert len({id(c) for c in (mine, *others)}) == 4
    assert default_context() is mine


def test_a_release_reaches_the_default_contexts_of_other_threads(rt):
    """Calls of a backward pass run on a thread of its own, and the step that releases runs on the main one. Their scratch is
    free again at that thread's next call, not while a call of it is under way."""
    from diopi_b200.runtime import default_context
    calls, replies = queue.Queue(), queue.Queue()

    def work():
        while calls.get():
            ctx = default_context()
            replies.put((scratch(rt, ctx), ctx.stats()["blocks"]))

    t = threading.Thread(target=work)
    t.start()
    try:
        def call():
            calls.put(True)
            return replies.get(timeout=60)
        first, _ = call()
        assert call()[0] != first                 # not released
        seen = set()
        for _ in range(20):
            default_context().release()
            got, blocks = call()
            seen.add(got)
        assert len(seen) == 1 and blocks == 2
    finally:
        calls.put(False)
        t.join()


@pytest.mark.gpu
def test_the_default_context_on_two_streams_at_once(built_libs):
    """Calls on torch's current stream, which changes from call to call, their scratch released each time."""
    from diopi_b200 import functions as F
    from diopi_b200.runtime import Context, default_context
    from test_gpu_quantized_cache import attention_inputs
    args = [[t.cuda() for t in attention_inputs([4000, 31, 700], seed=s)] for s in range(2)]
    wants = [F.quantized_paged_attention(*a, 0.1, ctx=Context()) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(w) for _ in range(50)] for w in wants]
    torch.cuda.synchronize()
    for i in range(50):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                F.quantized_paged_attention(*args[s], 0.1, out=outs[s][i])
                default_context().release()
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(o, wants[s]) for o in outs[s])


@pytest.mark.gpu
def test_a_capture_takes_the_scratch_of_the_stream_that_warmed_up(built_libs):
    """Nothing can be allocated while a stream is captured: the capture gets what another stream has released."""
    from diopi_b200 import functions as F
    from diopi_b200.runtime import Context
    from test_gpu_quantized_cache import attention_inputs
    args = [t.cuda() for t in attention_inputs([2000, 31, 700], seed=3)]
    ctx = Context()
    want = F.quantized_paged_attention(*args, 0.1, ctx=ctx)
    ctx.release()
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.set_stream(torch.cuda.current_stream())
        F.quantized_paged_attention(*args, 0.1, ctx=ctx, out=out)
    ctx.release()
    ctx.set_stream(torch.cuda.current_stream())
    allocs = ctx.stats()["device_allocs"]
    for _ in range(10):       # eager calls beside the replays: scratch of their own
        graph.replay()
        other = F.quantized_paged_attention(*args, 0.1, ctx=ctx)
        ctx.release()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)
        out.zero_()
    assert ctx.stats()["device_allocs"] == allocs + 1


@pytest.mark.gpu
def test_calls_beside_a_graph_of_their_context(built_libs):
    """The graph is replayed on another stream than the one it was captured on, where eager calls go on: they have scratch of their
    own. Graphs captured one after the other share theirs."""
    from diopi_b200 import functions as F
    from diopi_b200.runtime import Context
    from test_gpu_quantized_cache import attention_inputs
    args = [[t.cuda() for t in attention_inputs([4000, 31, 700], seed=s)] for s in range(2)]
    st, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(st):
        ctx = Context(st)
        wants = [F.quantized_paged_attention(*a, 0.1, ctx=Context(st)) for a in args]
        F.quantized_paged_attention(*args[0], 0.1, ctx=ctx)
        outs = [torch.empty_like(w) for w in wants]
        st.synchronize()
        graphs = []
        for _ in range(2):
            ctx.release()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=st):
                F.quantized_paged_attention(*args[0], 0.1, ctx=ctx, out=outs[0])
        ctx.release()
        assert ctx.stats()["blocks"] == 1
        eager = [torch.empty_like(wants[1]) for _ in range(40)]
        F.quantized_paged_attention(*args[1], 0.1, ctx=ctx, out=eager[0])
        assert ctx.stats()["blocks"] == 2
        torch.cuda.synchronize()
        for e in eager:
            ctx.release()
            F.quantized_paged_attention(*args[1], 0.1, ctx=ctx, out=e)
            with torch.cuda.stream(other):
                graphs[0].replay()
        torch.cuda.synchronize()
        assert ctx.stats()["blocks"] == 2
        assert torch.equal(outs[0], wants[0]) and all(torch.equal(e, wants[1]) for e in eager)
