"""Calls over caches that need a workspace, side by side: captured graphs on streams of their own, eager calls, threads."""

import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture
def ctx():
    """A context of its own: its workspaces are those of these calls."""
    from quantibbler_b200.gpu import GpuContext
    ctx = GpuContext.init()
    yield ctx
    torch.cuda.synchronize()
    ctx.close()


def make(ctx, g, dtype, n_seq, kv, rows, d):
    from quantibbler_b200.cache import KvCache
    shape = (n_seq, kv, rows, d)
    if dtype == "bfloat16":
        return KvCache(ctx, *(torch.randn(shape, device="cuda", generator=g).bfloat16() for _ in range(2)))
    codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
    return KvCache(ctx, *codes, *(torch.rand(shape[:3], device="cuda", generator=g) * 0.01 + 0.01 for _ in range(2)))


def calls(ctx, dtype):
    """[(bytes of workspace, a call that returns its output)] of a step, a step behind a prefix and a portion."""
    from quantibbler_b200 import _lib
    lib, g = _lib.lib(), torch.Generator(device="cuda").manual_seed(1)
    step, shared, long = make(ctx, g, dtype, 40, 2, 700, 128), make(ctx, g, dtype, 1, 2, 3000, 128), make(ctx, g, dtype, 2, 2, 4000, 128)
    q, many = (torch.randn(n, 8, 128, device="cuda", generator=g) for n in (40, 150))
    lens = torch.randint(0, 701, (40,), device="cuda", generator=g, dtype=torch.int32)
    ref = lambda c: ctypes.byref(c._c)  # noqa: E731
    return [(lib.qk_cache_attend_scratch(ref(step), 0, 40, 8), lambda: step.attend(q, lens)),
            (lib.qk_cache_attend_scratch(ref(step), 3000, 40, 8), lambda: step.attend(q, lens, prefix=shared, prefix_len=3000)),
            (lib.qk_cache_portion_scratch(ref(long), 3500, 0, 150, 8), lambda: long.portion(many, 1, 3500))]


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_graphs_and_eager_calls_at_once(ctx, dtype):
    """Three captured calls, replayed on three streams at once beside eager ones of the same on a fourth."""
    todo = calls(ctx, dtype)
    assert all(size > 0 for size, _ in todo)
    want = [call() for _, call in todo]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    graphs = []
    for stream, (_, call) in zip(streams, todo):
        ctx.set_stream(stream.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        graphs.append((stream, graph, out))
    ctx.set_stream(streams[3].cuda_stream)
    eager = []
    for _ in range(20):
        for stream, graph, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[3]):
            eager = [call() for _, call in todo]
    torch.cuda.synchronize()
    for w, e, (_, _, out) in zip(want, eager, graphs):
        assert torch.equal(out, w) and torch.equal(e, w)
    ctx.synchronize()


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_threads_whose_calls_need_more_and_more(ctx, dtype):
    """Three threads on streams of their own share a context: its workspace grows while the others' calls use it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    c = make(ctx, g, dtype, 2, 8, 4000, 128)
    sizes = (20, 40, 90, 150, 400)
    qs = [torch.randn(n, 32, 128, device="cuda", generator=g) for n in sizes]
    wants = [c.portion(q, 1, 3500) for q in qs]
    torch.cuda.synchronize()
    ctx.workspaces.clear()
    off = []

    def work(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for i in order * 5:
                got = c.portion(qs[i], 1, 3500)
                stream.synchronize()
                if not torch.equal(got, wants[i]):
                    off.append(sizes[i])

    threads = [threading.Thread(target=work, args=(o,)) for o in ([0, 1, 2, 3, 4], [0, 2, 1, 4, 3], [1, 0, 3, 2, 4])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not off and max(map(len, ctx.workspaces.values())) > 1


def test_a_workspace_is_memory_of_the_contexts_stream(ctx):
    """It is not taken from what the caller's stream has just given back (kernels of that stream may be using it still, and
    another thread's call may get to the workspace first)."""
    size, call = calls(ctx, "int8")[2]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.workspaces.clear()
    with torch.cuda.stream(side):
        freed = torch.empty(size, dtype=torch.uint8, device="cuda")
        begin, end = freed.data_ptr(), freed.data_ptr() + size
        del freed
        call()
    torch.cuda.synchronize()
    (kept,) = ctx.workspaces.values()
    assert kept[-1].numel() >= size and not (begin <= kept[-1].data_ptr() < end)
