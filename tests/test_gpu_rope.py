"""Norm and position rotation of query and key heads (omni_qk_norm_rope and
its gradient) against the formulas in 64 bits.

Bars, derived before the first run.  u is half a step of a type relative to
the value (finfo.eps / 2), u32 that of fp32.  An output is rounded once from
fp32, u |y|; its fp32 value is z cos + z' sin, where z = x r w carries the
errors of the mean of squares (D + 1 roundings of positive terms, halved by
the square root), the reciprocal root (one step, 2 u32) and two products, and
cos and sin err by 4 u32 (a 24-bit remainder, 2e-9 of the series, the
polynomials' roundings): (D / 2 + 12) u32 (|z| + |z'|) bounds it for every D
here with room.  A gradient adds the second mean, of g x over D terms:
(2 D + 30) u32 (|g| + mean |g x| |x|) r.  A weight gradient is a sum of n
terms in fp32 in an order of its own: at most n u32 sum |term|, and in
practice sqrt(n); 64 + sqrt(n) is taken, far above any run of at most a few
thousand additions that a lane makes.
"""
import math
from fractions import Fraction

import pytest
import torch

from tests import _data

gpu = pytest.mark.gpu
U32 = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _turn64(x, theta, pairs, R):
    """x (N, H, D) float64, theta (N, R / 2): the rotated x and |z| + |z'|."""
    y, mag = x.clone(), x.abs()
    c, s = theta.cos()[:, None], theta.sin()[:, None]
    lo, hi = (slice(0, R // 2), slice(R // 2, R)) if pairs == "halves" else (slice(0, R, 2), slice(1, R, 2))
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    mag[..., lo] = mag[..., hi] = a.abs() + b.abs()
    return y, mag


def _want(x, w, theta, pairs, R, eps, dy=None):
    """(y, bar on y, dx, bar on dx, dw, bar on dw) in float64."""
    D, u = x.shape[-1], _u(x.dtype)
    x = x.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if w is not None else torch.ones_like(x[..., :1])
    wd = w.double() if w is not None else torch.ones(D, dtype=torch.float64)
    y, mag = _turn64(x * r * wd, theta, pairs, R)
    ybar = u * y.abs() + (D / 2 + 12) * U32 * mag
    if dy is None:
        return y, ybar
    dz, dmag = _turn64(dy.double(), -theta, pairs, R)
    if w is None:
        return y, ybar, dz, u * dz.abs() + 12 * U32 * dmag, None, None
    g, xh = dz * wd, x * r
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    dxmag = r * (dmag * wd.abs() + (dmag * wd.abs() * xh.abs()).mean(-1, keepdim=True) * xh.abs())
    n = x.shape[0] * x.shape[1]
    dw = (dz * xh).sum((0, 1))
    dwbar = _u(w.dtype) * dw.abs() + (64 + math.sqrt(n) + D / 2) * U32 * (dmag * xh.abs()).sum((0, 1))
    return y, ybar, dx, u * dx.abs() + (2 * D + 30) * U32 * dxmag, dw, dwbar


def _close(got, want, bar, tag):
    err = (got.double().cpu() - want).abs()
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps    # half a step of a subnormal
    ratio = (err / (bar + tiny)).max().item() if err.numel() else 0.0
    print(f"[rope] {tag}: worst error / bar {ratio:.3f}", flush=True)
    ok = bool((err <= bar + tiny).all())
    assert ok, f"{tag}: {ratio}"


def _inputs(N, Hq, Hkv, D, dtype, seed, wdt=None):
    g = _data.gen(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(DT[dtype])  # noqa: E731
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(DT[wdt]) for _ in range(2)] if wdt else [None, None]
    return mk(N, Hq, D), mk(N, Hkv, D), mk(N, Hq, D), mk(N, Hkv, D), *w


def _theta(positions, rotary_dim, axes, base=10000.0):
    n = rotary_dim // 2
    f = torch.tensor([base ** (-i / n) for i in range(n)], dtype=torch.float64)
    return positions[torch.as_tensor(axes)].double().T * f


@gpu
@pytest.mark.parametrize("N,Hq,Hkv,D,dtype,wdt,R,pairs,first", [
    (1, 32, 8, 128, "bf16", "bf16", 128, "halves", 0),
    (64, 32, 8, 128, "bf16", "bf16", 128, "halves", 100000),
    (257, 7, 1, 128, "f16", "f32", 64, "halves", 5),
    (33, 16, 4, 32, "f32", "f32", 32, "neighbours", 3),
    (19, 5, 3, 64, "bf16", "f16", 32, "neighbours", -7),
    (13, 3, 2, 256, "f16", "f16", 256, "halves", 1 << 21),
    (9, 6, 1, 256, "f32", "bf16", 128, "halves", 1 << 40),
    (2500, 2, 2, 32, "bf16", "bf16", 16, "halves", 17),
    (41, 4, 4, 64, "f32", "f32", 64, "halves", 0),
    (70, 9, 3, 32, "f16", None, 32, "halves", 1 << 20),
    (70, 9, 3, 128, "bf16", None, 0, "halves", 1),
    (5, 2, 1, 256, "bf16", None, 224, "neighbours", 1),
])
def test_outputs_and_gradients(device, N, Hq, Hkv, D, dtype, wdt, R, pairs, first):
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    q, k, gq, gk, wq, wk = _inputs(N, Hq, Hkv, D, dtype, N + D, wdt)
    pos = (torch.arange(N) * 3 + first)[None]
    if first >= 1 << 40:
        # far positions: the product with a frequency has more than 64-bit floats
        # hold (2 pi / 8 itself is off by 2^-53, 1e-4 of a radian at 2^40), so the
        # angle is the exact product of the integer and the float, less whole turns
        freq = [2 * math.pi / 2 ** (i % 30 + 3) for i in range(R // 2)]
        rot = RotaryEmbedding(D, rotary_dim=R, inv_freq=freq, interleaved=pairs != "halves", device=device)
        turn = 2 * Fraction(31415926535897932384626433832795028841971, 10 ** 40)
        theta = torch.tensor([[float(int(p) * Fraction(f) % turn) for f in freq] for p in pos[0]], dtype=torch.float64)
    else:
        rot = RotaryEmbedding(D, rotary_dim=R, interleaved=pairs != "halves", device=device)
        theta = _theta(pos, R, [0] * (R // 2)) if R else torch.zeros(N, 0, dtype=torch.float64)
    leaves = [t.to(device).requires_grad_() for t in (q, k, wq, wk) if t is not None]
    y = qk_norm_rope(leaves[0], leaves[1], pos[0].to(device), rot, *(leaves[2:] or (None, None)), 1e-6)
    grads = torch.autograd.grad(y, leaves, (gq.to(device), gk.to(device)))
    again = torch.autograd.grad(qk_norm_rope(leaves[0], leaves[1], pos[0].to(device), rot, *(leaves[2:] or (None, None)), 1e-6),
                                leaves, (gq.to(device), gk.to(device)))
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "not the same on a second run"
    for i, (x, w, dy) in enumerate(((q, wq, gq), (k, wk, gk))):
        yw, yb, dx, dxb, dw, dwb = _want(x, w, theta, pairs, R, 1e-6, dy)
        _close(y[i].detach(), yw, yb, f"{'qk'[i]} out")
        _close(grads[i], dx, dxb, f"{'qk'[i]} grad")
        if w is not None:
            _close(grads[2 + i], dw, dwb, f"{'qk'[i]} weight grad")


@gpu
def test_gradient_against_differences(device):
    """Central differences of the kernel's own fp32 outputs: step h, truncation
    h^2 / 6 times a third derivative of order one, outputs off by 1e-6 of
    their size over h."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    q, k, gq, gk, wq, wk = (t.to(device) for t in _inputs(3, 2, 1, 32, "f32", 77, "f32"))
    rot = RotaryEmbedding(32, device=device)
    pos = torch.tensor([0, 5, 911], device=device)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(qk_norm_rope(*leaves[:2], pos, rot, *leaves[2:]), leaves, (gq, gk))
    h = 2.0 ** -7
    with torch.no_grad():
        def loss():
            a, b = qk_norm_rope(*leaves[:2], pos, rot, *leaves[2:])
            return (a.double() * gq.double()).sum() + (b.double() * gk.double()).sum()
        for t, g in zip(leaves, grads):
            for i in (0, t.numel() // 2 + 3, t.numel() - 1):
                old = t.view(-1)[i].item()
                t.view(-1)[i] = old + h
                hi = loss()
                t.view(-1)[i] = old - h
                lo = loss()
                t.view(-1)[i] = old
                assert abs((hi - lo).item() / (2 * h) - g.view(-1)[i].item()) < 2e-2 * max(1.0, abs(g.view(-1)[i].item()))


@gpu
@pytest.mark.parametrize("layout", ["fused", "bhtd", "every_second_head", "odd_start", "last_dim_step"])
def test_layouts(device, layout):
    """Strided inputs give what contiguous ones give, bit for bit."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, Hq, Hkv, D = 22, 6, 2, 64
    q, k, gq, gk, wq, wk = (t.to(device) for t in _inputs(N, Hq, Hkv, D, "bf16", 5, "bf16"))
    rot = RotaryEmbedding(D, device=device)
    pos = torch.arange(N, device=device) + 50
    want = qk_norm_rope(q, k, pos, rot, wq, wk)
    if layout == "bhtd":                           # two sequences of 11
        q4, k4 = (t.view(2, 11, -1, D).transpose(1, 2) for t in (q, k))
        got = qk_norm_rope(q4, k4, pos.view(2, 11), rot, wq, wk)
        assert got[0].shape == (2, Hq, 11, D) and got[0].is_contiguous()
        got = [t.transpose(1, 2).reshape(N, -1, D) for t in got]
        one = qk_norm_rope(q4, k4, pos[:11], rot, wq, wk)[0]          # one row of positions for both
        assert torch.equal(one[0], q4.new_tensor(0) + want[0].view(2, 11, Hq, D)[0].transpose(0, 1))
    else:
        if layout == "fused":
            buf = torch.cat([q.reshape(N, -1), k.reshape(N, -1), k.reshape(N, -1)], 1)
            qs, ks = buf[:, :Hq * D].view(N, Hq, D), buf[:, Hq * D:(Hq + Hkv) * D].view(N, Hkv, D)
        elif layout == "every_second_head":
            qs, ks = (torch.stack([t, t + 1], 2).view(N, -1, D)[:, ::2] for t in (q, k))
        elif layout == "odd_start":                # rows off 16 bytes: copied first
            qs, ks = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k))
        else:
            qs, ks = (torch.stack([t, t], -1)[..., 0] for t in (q, k))
        got = qk_norm_rope(qs, ks, pos, rot, wq, wk)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
def test_axes(device):
    """Three position axes: sections and pair_axes agree, and each pair turns by its own axis."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, D = 30, 128
    q, k, _, _, _, _ = _inputs(N, 4, 2, D, "f16", 8)
    pos = torch.stack([torch.arange(N) // 6, torch.arange(N) // 3 % 2, torch.arange(N) % 3 + 1000])
    axes = [0] * 16 + [1] * 24 + [2] * 24
    a = qk_norm_rope(q.to(device), k.to(device), pos.to(device), RotaryEmbedding(D, sections=(16, 24, 24), device=device))
    b = qk_norm_rope(q.to(device), k.to(device), pos.to(device), RotaryEmbedding(D, pair_axes=axes, device=device))
    for x, y, z in zip((q, k), a, b):
        assert torch.equal(y, z)
        _close(y, *_want(x, None, _theta(pos, D, axes), "halves", D, 0.0), "axes")
    # one row of positions for every axis is the text rotation
    text = qk_norm_rope(q.to(device), k.to(device), pos[2].to(device), RotaryEmbedding(D, sections=(16, 24, 24), device=device))
    plain = qk_norm_rope(q.to(device), k.to(device), pos[2].int().to(device), RotaryEmbedding(D, device=device))
    assert all(torch.equal(x, y) for x, y in zip(text, plain))


@gpu
def test_in_place_and_out(device):
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, Hq, Hkv, D = 50, 8, 2, 128
    q, k, _, _, wq, wk = (t.to(device) for t in _inputs(N, Hq, Hkv, D, "bf16", 15, "f32"))
    rot, pos = RotaryEmbedding(D, device=device), torch.arange(N, device=device)
    want = qk_norm_rope(q, k, pos, rot, wq, wk)
    buf = torch.cat([q.reshape(N, -1), k.reshape(N, -1), k.reshape(N, -1)], 1)
    qs, ks = buf[:, :Hq * D].view(N, Hq, D), buf[:, Hq * D:(Hq + Hkv) * D].view(N, Hkv, D)
    tail = buf[:, (Hq + Hkv) * D:].clone()
    got = qk_norm_rope(qs, ks, pos, rot, wq, wk, out=(qs, ks))
    assert got[0] is qs and torch.equal(qs, want[0]) and torch.equal(ks, want[1])
    assert torch.equal(buf[:, (Hq + Hkv) * D:], tail)
    buf = torch.cat([q.reshape(N, -1), k.reshape(N, -1)], 1)
    qs, ks = (t.unflatten(0, (2, 25)).transpose(1, 2) for t in (buf[:, :Hq * D].view(N, Hq, D), buf[:, Hq * D:].view(N, Hkv, D)))
    qk_norm_rope(qs, ks, pos.view(2, 25), rot, wq, wk, out=(qs, ks))       # (2, heads, 25, D)
    assert all(torch.equal(t.transpose(1, 2).reshape(w.shape), w) for t, w in zip((qs, ks), want))
    with pytest.raises(ValueError, match="overlap"):
        qk_norm_rope(q[1:], k[1:], pos[1:], rot, wq, wk, out=(q[:-1], torch.empty_like(k[1:])))
    with pytest.raises(ValueError, match="overlap itself"):
        qk_norm_rope(q, k, pos, rot, wq, wk, out=(torch.empty(N * D + Hq * D, device=device, dtype=q.dtype).as_strided((N, Hq, D), (D, D, 1)), k))
    with pytest.raises(ValueError, match="gradient"):
        qk_norm_rope(q, k, pos, rot, wq.clone().requires_grad_(), wk, out=(q, k))
    with pytest.raises(ValueError, match="gradient"):
        qk_norm_rope(q, k, pos, rot, wq, wk, out=(torch.empty_like(q, requires_grad=True), torch.empty_like(k)))


@gpu
def test_far_offsets_and_version(device):
    """Token strides of 2 MB: the last tokens lie past 2^32 bytes.  Writing in
    place is seen by a graph that saved the tensor."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, Hq, Hkv, D = 2200, 4, 2, 64
    q, k, gq, gk, wq, wk = (t.to(device) for t in _inputs(N, Hq, Hkv, D, "bf16", 16, "bf16"))
    rot, pos = RotaryEmbedding(D, device=device), torch.arange(N, device=device)
    want = qk_norm_rope(q, k, pos, rot, wq, wk)
    buf = torch.empty(N, 1 << 20, dtype=torch.bfloat16, device=device)
    qs, ks = buf[:, :Hq * D].view(N, Hq, D), buf[:, -Hkv * D:].view(N, Hkv, D)
    qs.copy_(q)
    ks.copy_(k)
    assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(qs, ks, pos, rot, wq, wk), want))
    before = qs._version
    qk_norm_rope(qs, ks, pos, rot, wq, wk, out=(qs, ks))
    assert torch.equal(qs, want[0]) and torch.equal(ks, want[1]) and qs._version > before


@gpu
def test_broadcast_inputs_and_gradients(device):
    """One key head spread over many and output gradients of one value: the bits of their copies."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, D = 37, 64
    q, k, _, _, wq, wk = (t.to(device) for t in _inputs(N, 4, 1, D, "bf16", 52, "f32"))
    rot, pos, one = RotaryEmbedding(D, device=device), torch.arange(N, device=device), q[:1, :1, :1]
    leaf = k.clone().requires_grad_()
    args = [q.clone().requires_grad_(), leaf.expand(N, 3, D), wq.requires_grad_(), wk.requires_grad_()]
    y = qk_norm_rope(*args[:2], pos, rot, *args[2:])
    grads = torch.autograd.grad(y, args, (one.expand(N, 4, D), one.expand(N, 3, D)), retain_graph=True)
    copies = [t.detach().contiguous().requires_grad_() for t in args]
    want = qk_norm_rope(*copies[:2], pos, rot, *copies[2:])
    ref = torch.autograd.grad(want, copies, (one.expand(N, 4, D).contiguous(), one.expand(N, 3, D).contiguous()))
    assert all(torch.equal(a.detach(), b.detach()) for a, b in zip((*y, *grads), (*want, *ref)))
    back, = torch.autograd.grad(y, [leaf], (one.expand(N, 4, D), one.expand(N, 3, D)))
    assert torch.equal(back, ref[1].sum(1, keepdim=True))


@gpu
def test_copied_rotary_embedding(device):
    """A copy holds its own frequencies and reads no others."""
    import copy

    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    q, k, *_ = (t.to(device) for t in _inputs(20, 4, 2, 64, "bf16", 51, "bf16"))
    pos = torch.arange(20, device=device)
    rot = RotaryEmbedding(64, device=device)
    other = copy.deepcopy(rot)
    want = qk_norm_rope(q, k, pos, rot)
    rot.turns.zero_()
    assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(q, k, pos, other), want))
    assert torch.equal(qk_norm_rope(q, k, pos, rot)[0], q)


@gpu
def test_zero_rows_and_special_values(device):
    """No tokens give no outputs (and zero weight gradients); a row of zeros
    stays zero; NaN and infinity stay in their own head."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    rot = RotaryEmbedding(64, device=device)
    w = torch.ones(64, device=device, requires_grad=True)
    w2 = torch.ones(64, device=device, requires_grad=True)
    e = torch.empty(0, 4, 64, device=device)
    y = qk_norm_rope(e, e[:, :2], torch.empty(0, dtype=torch.int32, device=device), rot, w, w2)
    assert y[0].shape == (0, 4, 64) and y[1].shape == (0, 2, 64)
    gw = torch.autograd.grad(y, (w, w2), (e, e[:, :2]))
    assert all(bool((g == 0).all()) for g in gw)
    x = torch.randn(6, 4, 64, device=device)
    x[2, 1] = 0
    x[3, 2, 5] = float("nan")
    x[4, 0, 7] = float("inf")
    y, _ = qk_norm_rope(x, x, torch.arange(6, device=device), rot, w.detach(), w.detach())
    assert bool((y[2, 1] == 0).all())
    bad = ~torch.isfinite(y).all(-1)
    want = torch.zeros(6, 4, dtype=torch.bool, device=device)
    want[3, 2] = want[4, 0] = True
    assert torch.equal(bad, want)


@gpu
def test_capture_and_other_stream(device):
    """Captured with its gradient and replayed with new values, refused while an
    eager graph of the same leaves is alive; and on a stream of its own."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    q, k, gq, gk, wq, wk = (t.to(device) for t in _inputs(40, 8, 2, 128, "bf16", 25, "bf16"))
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    rot, pos = RotaryEmbedding(128, device=device), torch.arange(40, device=device)

    def step():
        y = qk_norm_rope(*leaves[:2], pos, rot, *leaves[2:])
        return (*y, *torch.autograd.grad(y, leaves, (gq, gk)))

    alive = qk_norm_rope(*leaves[:2], pos, rot, *leaves[2:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    shape = alive[0].shape
    del alive, first, want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [t.detach() for t in step()]
    for i in range(3):
        with torch.no_grad():
            q.mul_(-1.5)
            pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        want = [t.detach() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"
    assert shape == q.shape


def test_refusals_of_the_rotary_embedding():
    from omnistack_rs.kernels.rope import RotaryEmbedding
    for kw in (dict(head_dim=96), dict(rotary_dim=12), dict(rotary_dim=256), dict(base=0.0), dict(base=float("inf")),
               dict(inv_freq=[1.0] * 63), dict(inv_freq=[float("nan")] * 64), dict(sections=(10, 10)),
               dict(sections=(-1, 65)), dict(pair_axes=[0] * 63), dict(pair_axes=[-1] * 64),
               dict(sections=(64,), pair_axes=[0] * 64), dict(pair_axes=[256] * 64)):
        with pytest.raises(ValueError):
            RotaryEmbedding(**{"device": "cpu", **kw})


def test_refusals_of_the_call():
    """Checked before any device work: on CPU tensors the last check is the device's."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    rot = RotaryEmbedding(64, device="cpu")
    q, k, pos, w = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64), torch.arange(5), torch.ones(64)
    with pytest.raises(RuntimeError, match="HIP"):
        qk_norm_rope(q, k, pos, rot, w, w)
    bad = [((q[0], k[0], pos, rot), {}), ((q, k[:4], pos, rot), {}), ((q[..., :32], k[..., :32], pos, rot), {}),
           ((q, k.half(), pos, rot), {}), ((q.double(), k.double(), pos, rot), {}), ((q, k, pos.float(), rot), {}), ((q, k, pos[:4], rot), {}),
           ((q, k, pos, rot, w), {}), ((q, k, pos, rot, w, w[:32]), {}), ((q, k, pos, rot, w, w.half()), {}),
           ((q, k, pos, rot, w, w, -1.0), {}), ((q, k, pos, rot, w, w, float("nan")), {}),
           ((q.half(), k.half(), pos, RotaryEmbedding(64, rotary_dim=24, device="cpu")), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            qk_norm_rope(*args, **kw)
    with pytest.raises(TypeError):
        qk_norm_rope(q, k, pos, None)


def test_folded():
    from omnistack_rs.kernels.rope import folded
    x = torch.zeros(4, 6, 8)
    assert not any(folded(t) for t in (x, x.transpose(0, 1), x[:, ::2], x[:1].transpose(0, 2), x[:0], torch.zeros(())))
    assert folded(x[:1].expand(4, 6, 8)) and folded(x[:, :1].expand(4, 6, 8))
    assert folded(x.view(-1).as_strided((4, 6, 8), (8, 8, 1))) and folded(x.view(-1).as_strided((4, 6, 8), (48, 4, 1)))


def test_overlap():
    from omnistack_rs.kernels.rope import overlap
    D, row = 8, (3 + 2 + 2) * 8
    buf = torch.zeros(10 * row)
    q, k = buf.view(10, 7, D)[:, :3], buf.view(10, 7, D)[:, 3:5]
    assert not overlap(q, k) and not overlap(k, q) and overlap(q, q) and overlap(q[1:], q[:-1]) and overlap(buf.view(10, 7, D)[:, 2:4], k)
    q4, k4 = (t.unflatten(0, (2, 5)).transpose(1, 2) for t in (q, k))     # (2, heads, 5, D)
    assert not overlap(q4, k4) and not overlap(k4, q4) and overlap(q4, q4) and overlap(q4[:1], q4) and overlap(q4, q4[:, 1:])
    assert not overlap(q4[:1], k4[1:]) and not overlap(q[:1], k[:1]) and not overlap(q, torch.zeros(10, 3, D))
    h = buf[:10 * 3 * D].view(3, 10, D).transpose(0, 1)                   # heads outermost: not told apart
    assert overlap(h, h[:, 1:]) and not overlap(h[:, :1], h[:, 1:])


def test_turns_are_the_frequencies():
    """Fractions of a turn: round(f / 2 pi 2^64), negative frequencies by wrap-around."""
    from omnistack_rs.kernels.rope import RotaryEmbedding
    rot = RotaryEmbedding(32, inv_freq=[2 * math.pi * x for x in (0.5, 0.25, 0.125, -0.25)] + [1.0] * 12, device="cpu")
    t = [int(x) % 2 ** 64 for x in rot.turns]
    for got, want in zip(t[:4], (2 ** 63, 2 ** 62, 2 ** 61, 2 ** 64 - 2 ** 62)):
        assert abs(got - want) < 2 ** 12            # the double 2 pi x is off by 2^-53 of itself
    assert abs(t[4] / 2 ** 64 - 1 / (2 * math.pi)) < 1e-16


def test_native_refusals():
    """The C entry points check sizes, alignment and NULLs before any device work."""
    import ctypes
    from omnistack_rs import _lib
    L = _lib.lib()
    s = (ctypes.c_int64 * 3)(0, 64, 64)
    odd = (ctypes.c_int64 * 3)(0, 63, 64)

    def call(q=4096, qs=s, dtype=0, D=64, R=64, wq=None, wk=None, eps=1e-6, pos=4096, B=1, T=2):
        return L.omni_qk_norm_rope(q, qs, 8192, s, dtype, B, T, 1, 1, D, pos, 0, s, 4096, 4096, R, 0, wq, wk, 0, eps,
                                   4096, s, 8192, s, None)
    for kw, msg in ((dict(D=48), "head_dim"), (dict(R=12), "rotary_dim"), (dict(R=72), "rotary_dim"), (dict(dtype=3), "dtype"),
                    (dict(q=4100), "16 bytes"), (dict(qs=odd), "16 bytes"), (dict(q=None), "NULL"), (dict(wq=4096), "together"),
                    (dict(wq=4097, wk=4096), "aligned"), (dict(wq=4096, wk=4096, eps=-1.0), "eps"), (dict(pos=None), "NULL"),
                    (dict(B=-1), "shape"), (dict(B=1 << 40, T=1 << 40), "large")):
        assert call(**kw) == _lib.OMNI_EINVAL and msg in _lib.last_error(), (kw, _lib.last_error())
    assert call(B=0) == 0 and call(T=0, q=None) == 0
    assert L.omni_qk_norm_rope_backward_workspace_size(128) == 1024 * 2 * 128 * 4
    rc = L.omni_qk_norm_rope_backward(4096, s, 4096, s, 0, 1, 2, 1, 1, 64, 4096, 0, s, 4096, 4096, 64, 0, 4096, 4096, 0, 1e-6,
                                      4096, s, 4096, s, 4096, s, 4096, s, 4096, 4096, None, 0, None)
    assert rc == _lib.OMNI_EWORKSPACE and "workspace" in _lib.last_error()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("R", [0, 32])
def test_dims_behind_the_rotation_are_copies(device, dtype, pairs, R):
    """Without a norm the dims behind rotary_dim keep their bits, infinities,
    NaN and zeros' signs among them, and so do their gradients; the dims that
    turn are those of ordinary neighbours."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, D = 23, 64
    q, k, gq, gk, _, _ = (t if t is None else t.to(device) for t in _inputs(N, 4, 2, D, dtype, 81))
    rot = RotaryEmbedding(D, rotary_dim=R, interleaved=pairs != "halves", device=device)
    pos = torch.arange(N, device=device) + 7
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    y = qk_norm_rope(*leaves, pos, rot)
    clean = [t.detach() for t in (*y, *torch.autograd.grad(y, leaves, (gq, gk)))]
    bad = [float("inf"), float("-inf"), float("nan"), -0.0]
    for t in (q, k, gq, gk):
        for i, x in enumerate(bad * 2):
            t[i::5, i % 2, R + 3 * i + 1] = x
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    y = qk_norm_rope(*leaves, pos, rot)
    got = [t.detach() for t in (*y, *torch.autograd.grad(y, leaves, (gq, gk)))]
    bits = torch.int32 if dtype == "f32" else torch.int16
    for g, c, x, name in zip(got, clean, (q, k, gq, gk), ("q", "k", "dq", "dk")):
        assert torch.equal(g[..., :R].view(bits), c[..., :R].view(bits)), name
        assert torch.equal(g[..., R:].contiguous().view(bits), x[..., R:].contiguous().view(bits)), name


@gpu
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_norm_with_an_infinity_behind_the_rotation(device, pairs):
    """The head's factor is 0 then: its finite dims are zeros, and only the
    infinite one is NaN."""
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    N, D, R = 9, 64, 32
    q, k, _, _, wq, wk = (t.to(device) for t in _inputs(N, 2, 1, D, "bf16", 82, "f32"))
    rot, pos = RotaryEmbedding(D, rotary_dim=R, interleaved=pairs != "halves", device=device), torch.arange(N, device=device)
    want = qk_norm_rope(q, k, pos, rot, wq, wk)
    for at in (R, R + 5, D - 1):
        x = q.clone()
        x[4, 1, at] = float("inf")
        got = qk_norm_rope(x, k, pos, rot, wq, wk)
        assert torch.equal(got[1], want[1])
        row = got[0][4, 1].clone()
        assert bool(torch.isnan(row[at])), at
        row[at] = 0
        assert bool((row == 0).all()), at
        got[0][4, 1] = want[0][4, 1]
        assert torch.equal(got[0], want[0])


def test_forward_mode_is_refused():
    """A dual tensor wants a derivative that the kernels do not form: refused
    before any device work, with and without gradients; the same numbers
    without a tangent get as far as the device check."""
    from torch.autograd import forward_ad
    from omnistack_rs.kernels.rope import RotaryEmbedding, _QKNormRope, qk_norm_rope
    rot, pos = RotaryEmbedding(64, device="cpu"), torch.arange(5)
    q, k, w = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64), torch.ones(64)
    with forward_ad.dual_level():
        for i in range(4):
            for grad in (False, True):
                args = [q, k, w, w]
                args[i] = forward_ad.make_dual(args[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    qk_norm_rope(*args[:2], pos, rot, *args[2:])
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    qk_norm_rope(*args[:2], pos, rot, *args[2:])
        dual = forward_ad.make_dual(q.clone(), torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qk_norm_rope(dual[1:], k[1:], pos[1:], rot)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qk_norm_rope(q, k, pos, rot, out=(dual, k))
        with pytest.raises(RuntimeError, match="HIP"):
            qk_norm_rope(q, k, pos, rot, w, w)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="HIP"):
            qk_norm_rope(dual, k, pos, rot)
        with pytest.raises(NotImplementedError, match="gradient has no forward-mode"):      # a tangent of the gradient
            _QKNormRope.backward(None, dual, k)
