"""Memory of a context whose calls were captured into a graph: what a graph writes when it is replayed is nobody else's."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_token_graphs import same, state, work  # noqa: E402


def capture(ctx, side, s):
    with torch.cuda.stream(side):
        work(ctx, s)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = work(ctx, s)
    return g, out


class Held:
    """Memory of the context that lives until it is given back (kdec_malloc), as a float tensor."""

    def __init__(self, ctx, n):
        from brosoundml_amd import native
        self.ctx, self.n, self.p = ctx, n, ctypes.c_void_p()
        ctx.call("kdec_malloc", 4 * n, ctypes.byref(self.p))
        self.hip = native.lib()

    @property
    def __cuda_array_interface__(self):
        return {"shape": (self.n,), "typestr": "<f4", "data": (self.p.value, False), "version": 2}

    def tensor(self):
        return torch.as_tensor(self, device=f"cuda:{self.ctx.device}")

    def free(self):
        self.ctx.call("kdec_free", self.p)


def test_memory_held_by_others_is_not_a_graphs():
    """After a capture, memory of many sizes (the pooled workspaces' among them, which a request of less than their size may
    get) is held, filled and still what it was after replays; the graph gives what it gave."""
    from brosoundml_amd import native
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    s = state(6, t=5000)
    want = [t.clone() for t in work(native.Context(0), state(6, t=5000))]
    torch.cuda.synchronize()
    g, out = capture(ctx, side, s)
    held = [Held(ctx, n) for n in [1 << b for b in range(6, 23)] * 3]
    views = [h.tensor() for h in held]
    with torch.cuda.stream(side):
        for i, v in enumerate(views):
            v.fill_(float(i + 1))
        for _ in range(3):
            g.replay()
            assert same(work(ctx, s), want)
    side.synchronize()
    assert same(out, want)
    for i, v in enumerate(views):
        assert (v == i + 1).all(), i
    del views
    for h in held:
        h.free()
    with torch.cuda.stream(side):
        g.replay()
    side.synchronize()
    assert same(out, want)


def test_memory_held_before_a_capture_stays_apart():
    """Memory that is held during a capture is not one of its workspaces, and given back later may serve the context's calls."""
    from brosoundml_amd import native
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    s = state(7)
    want = [t.clone() for t in work(native.Context(0), state(7))]
    torch.cuda.synchronize()
    held = [Held(ctx, 1 << 18) for _ in range(4)]
    views = [h.tensor() for h in held]
    with torch.cuda.stream(side):
        for v in views:
            v.fill_(3.0)
    g, out = capture(ctx, side, s)
    with torch.cuda.stream(side):
        g.replay()
    side.synchronize()
    assert same(out, want) and all((v == 3).all() for v in views)
    del views
    for h in held:
        h.free()
    with torch.cuda.stream(side):
        for _ in range(2):
            assert same(work(ctx, s), want)
            g.replay()
    side.synchronize()
    assert same(out, want)


def test_a_capture_reuses_what_it_gave_back():
    """Memory that is asked for and given back within a capture serves its next request, as outside of one, but no later
    capture's, whose memory outlives the first graph's replays."""
    from brosoundml_amd import native
    n = 1 << 22  # more than any of this context's other blocks
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    Held(ctx, n).free()  # one block for them all
    held, graphs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        if i:
            Held(ctx, n).free()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for _ in range(3):
                h = Held(ctx, n)
                h.tensor().fill_(float(i))
                h.free()
            held.append(Held(ctx, n))
            held[i].tensor().fill_(float(i + 5))
        graphs.append(g)
    assert held[0].p.value != held[1].p.value
    with torch.cuda.stream(side):
        for g in graphs + graphs:
            g.replay()
    side.synchronize()
    for i, h in enumerate(held):
        assert (h.tensor() == i + 5).all()
        h.free()


def test_calls_on_another_stream_stay_apart():
    """A context that moved to another stream makes its calls there while the graph is replayed on its own."""
    from brosoundml_amd import native
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    s, s2 = state(9, t=5000), state(10, t=5000)
    want, want2 = ([t.clone() for t in work(native.Context(0), state(i, t=5000))] for i in (9, 10))
    torch.cuda.synchronize()
    g, out = capture(ctx, side, s)
    ctx.call("kdec_set_stream", other.cuda_stream)
    ctx.stream = other
    got = []
    for _ in range(8):
        with torch.cuda.stream(side):
            g.replay()
        with torch.cuda.stream(other):
            got.append(work(ctx, s2))
    torch.cuda.synchronize()
    assert same(out, want) and all(same(o, want2) for o in got)


def test_a_capture_while_calls_are_timed():
    """With the context's timing on, captured calls are not timed (their events would never be read), and later calls work."""
    from brosoundml_amd import native
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    s = state(8)
    want = [t.clone() for t in work(native.Context(0), state(8))]
    torch.cuda.synchronize()
    ctx.profile(True)
    g, out = capture(ctx, side, s)
    with torch.cuda.stream(side):
        g.replay()
    side.synchronize()
    times = ctx.profile_read()
    with torch.cuda.stream(side):
        got = work(ctx, s)
        g.replay()
    side.synchronize()
    assert same(got, want) and same(out, want)
    again = ctx.profile_read()
    ctx.profile(False)
    for name in ("embed", "resnorm", "cache", "attn"):
        assert times[name]["ms"] > 0 and again[name]["launches"] == 2 * times[name]["launches"]
