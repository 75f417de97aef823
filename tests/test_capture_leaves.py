"""A gradient under graph capture while an eager graph of the same leaves is
alive, the leaves being behind views and products: refused, since the captured
backward pass would make the capture wait for the default stream."""
import gc

import pytest
import torch

from tests import _data


class _Op(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y):
        return x * 2, y * 2

    @staticmethod
    def backward(ctx, g, h):
        return g * 2, h * 2


@pytest.fixture
def streams(monkeypatch):
    """_lib with a current stream of the test's choice, which is captured or not."""
    from omnistack_rs import _lib
    now = dict(stream=0, capturing=False)
    monkeypatch.setattr(_lib, "stream_of", lambda device: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])

    def call(x, y, **kw):
        now.update(kw)
        out = _Op.apply(x, y)
        _lib.mark_leaves(torch.device("cpu"), out[0].grad_fn)
        return out
    return call


def _behind(leaf):
    """Through a view, a product, an earlier operator and a branch."""
    return (leaf.view(2, 3).t() * 3).reshape(-1) + leaf


def test_leaves_behind_other_nodes(streams):
    a, b, c = (torch.ones(6, requires_grad=True) for _ in range(3))
    alive = streams(_behind(a), b.detach(), stream=0, capturing=False)
    with pytest.raises(RuntimeError, match="still alive"):
        streams(c * 1, _behind(_behind(a)), stream=7, capturing=True)
    # other leaves, or no capture
    streams(_behind(c), _behind(b), stream=7, capturing=True)
    streams(_behind(a), b * 2, stream=7, capturing=False)
    del alive
    streams(_behind(a), b * 2, stream=7, capturing=True)


def test_the_eager_graph_counts_while_its_outputs_live(streams):
    a, b = (torch.ones(6, requires_grad=True) for _ in range(2))
    x = streams(_behind(a), b * 1, stream=0, capturing=False)[0] + 1          # kept by what came of them
    x.sum().backward()
    a.grad = b.grad = None
    with pytest.raises(RuntimeError, match="still alive"):
        streams(b.view(3, 2), a.detach(), stream=7, capturing=True)
    del x
    streams(b.view(3, 2), a.detach(), stream=7, capturing=True)
    # a node's context may outlive its graph
    out = streams(_behind(a), b * 1, stream=0, capturing=False)
    context = out[0].grad_fn
    del out
    streams(_behind(a), b * 1, stream=7, capturing=True)
    del context
    # a graph of another stream than the default one is joined by the engine
    side = streams(_behind(a), b * 1, stream=5, capturing=False)
    streams(_behind(a), b * 1, stream=7, capturing=True)
    del side


@pytest.mark.gpu
def test_capture_with_projections(device):
    """Query and key heads as products of leaves, both operators one after
    another: refused while the eager outputs live, then captured and replayed."""
    from omnistack_rs.attention import prompt_attention
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, Hq, Hkv, D = 90, 4, 2, 64
    g = _data.gen(90)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(device)  # noqa: E731
    x, w, wn, do = mk(N, (Hq + 2 * Hkv) * D), mk(N, (Hq + 2 * Hkv) * D), mk(D), mk(N, Hq, D)
    w.requires_grad_()
    rot, pos = RotaryEmbedding(D, device=device), torch.arange(N, device=device)
    cu = torch.tensor([0, 60, N], dtype=torch.int32, device=device)

    def forward():
        q, k, v = (x * w).view(N, -1, D).split([Hq, Hkv, Hkv], 1)
        q, k = qk_norm_rope(q, k, pos, rot, wn, wn)
        return prompt_attention(q, k, v, cu, validate=False)

    def step():
        o = forward()
        return o.detach(), *torch.autograd.grad(o, [w], do)

    alive = forward()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    gc.collect()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(-1.25)
            pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {i}"


def test_other_threads_may_build_graphs_meanwhile(streams):
    """The walk takes a snapshot: graphs that other threads make and drop during it are no error."""
    import threading
    a, b = (torch.ones(6, requires_grad=True) for _ in range(2))
    keep = [streams(_behind(a), b * 1, stream=0) for _ in range(200)]
    stop = threading.Event()

    def churn():
        from omnistack_rs import _lib
        while not stop.is_set():
            out = _Op.apply(a * 1, b * 1)
            _lib._default_nodes.add(_lib.weakref.ref(out[0].grad_fn, _lib._default_nodes.discard))

    t = threading.Thread(target=churn)
    t.start()
    try:
        for _ in range(20):
            with pytest.raises(RuntimeError, match="still alive"):
                streams(_behind(a), b * 1, stream=7, capturing=True)
    finally:
        stop.set()
        t.join()
    assert len(keep) == 200
