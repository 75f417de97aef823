"""Attention of packed prompts (omni_prompt_attn) and its gradient against the
definition in 64 bits.

Bars, derived before the first run.  u is half a step of the inputs' type,
u32 that of fp32.  Scores are fp32 sums of exact products: each is off by at
most (D + 2) u32 |scale| sum |q||k| <= X, an absolute error in the exponent, so
a probability is off by a factor within 1 +- (2 X + 2^-20) (its own error, the
row sum's and the exponential's).  A probability is then rounded to the
inputs' type, u p, before the product with v; row sums take the rounded, so
that the weights' errors d_s, |d_s| <= u p, leave sum_s d_s (v - o), at most
u sum_s p |v| + u |o|.
So |o - o'| <= (u + 2 X + 2^-20) sum_s p |v| + 2 u |o|.
Backward, with e = 2 X + 2^-20 + u for a rounded probability: dv is off by
e sum p |g| + u |dv|.  dp - delta is an fp32 sum of D products, and delta comes
from the rounded output: off by Y = (u + D u32) (|g| . |o| + sum_d |g||v|) + |g| . |o - o'|;
ds = p (dp - delta) by p Y + (e + u) |ds|; dq and dk by |scale| times the sum of
that with |k| or |q|, and u of themselves.  f16 subnormals: probabilities are
held times 2^7 at least, ds at least 2^-26 of its bound 2 max|g| max|v|.  bf16 goes
as far down as fp32, whose exponential gives 0 below the smallest normal, and
whose products do: 2^-126 a probability and a ds more (at scale 3 a key's
gradient was 0 for 1.9e-38, all of its terms of that size, before this term was
in the bar).
"""
import math

import pytest
import torch

from tests import _data

gpu = pytest.mark.gpu
U32 = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _cu(lengths, extra=0):
    c = [0]
    for n in lengths:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32), c[-1] + extra


def _inputs(N, Hq, Hkv, D, dtype, seed, gain=1.0):
    g = _data.gen(seed)
    mk = lambda h: torch.randn(N, h, D, generator=g)  # noqa: E731
    return (mk(Hq) * gain).to(DT[dtype]), mk(Hkv).to(DT[dtype]), mk(Hkv).to(DT[dtype]), mk(Hq).to(DT[dtype])


def _visible(x, seen):
    """0 where not seen, whatever stands there."""
    return torch.where(seen, x, torch.zeros_like(x))


def _want(q, k, v, cu, causal, scale, do=None):
    """Outputs, gradients and their bars in float64 on the inputs' device, by
    sequence and head; hidden keys and rows count for nothing, NaN or not."""
    u, D, G = torch.finfo(q.dtype).eps / 2, q.shape[2], q.shape[1] // k.shape[1]
    q64, k64, v64 = q.double(), k.double(), v.double()
    o, ob = torch.zeros_like(q64), torch.zeros_like(q64)
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    r = dict(o=(o, ob), lse=lse)
    if do is not None:
        g64 = do.double()
        for n, t in (("dq", q64), ("dk", k64), ("dv", v64)):
            r[n] = (torch.zeros_like(t), torch.zeros_like(t))
        n = int(cu[-1])
        tiny = 2.0 ** -25 * (g64[:n].norm(dim=-1).max() * v64[:n].norm(dim=-1).max()) if n and q.dtype == torch.float16 else 0.0
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        if a == b:
            continue
        see = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril()
        for h in range(q.shape[1]):
            Q, K, V = q64[a:b, h], k64[a:b, h // G], v64[a:b, h // G]
            s = torch.where(see, Q @ K.T * scale, -math.inf)
            p = torch.softmax(s, -1)
            l = torch.logsumexp(s, -1)
            X = (D + 2) * U32 * abs(scale) * _visible(Q.abs() @ K.abs().T, see)
            e = u + 2 * X.amax(-1, keepdim=True) + 2.0 ** -20
            O = p @ V
            o[a:b, h], lse[h, a:b] = O, l
            pmin = 2.0 ** -126 if q.dtype == torch.bfloat16 else 2.0 ** -31
            ob[a:b, h] = 2 * u * O.abs() + e * (p @ V.abs()) + pmin * (see.double() @ V.abs())
            if do is None:
                continue
            g = g64[a:b, h]
            dp = g @ V.T
            delta = (g * O).sum(-1, keepdim=True)
            Y = (u + D * U32) * (g.abs() @ V.abs().T + (g.abs() * O.abs()).sum(-1, keepdim=True)) + \
                (g.abs() * ob[a:b, h]).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            dsb = p * Y + (e + u) * ds.abs() + (tiny + 2.0 ** -126 * (1 + (dp - delta).abs())) * see.double()
            r["dq"][0][a:b, h] = ds @ K * scale
            r["dq"][1][a:b, h] = dsb @ K.abs() * abs(scale) + u * (ds @ K * scale).abs()
            r["dk"][0][a:b, h // G] += ds.T @ Q * scale
            r["dk"][1][a:b, h // G] += dsb.T @ Q.abs() * abs(scale)
            r["dv"][0][a:b, h // G] += p.T @ g
            pm = 2.0 ** -126 if q.dtype == torch.bfloat16 else 2.0 ** -38
            r["dv"][1][a:b, h // G] += (p * e).T @ g.abs() + pm * (see.double().T @ g.abs())
    if do is not None:
        for n in ("dk", "dv"):
            r[n][1].add_(u * r[n][0].abs())
    return r


def _close(got, want, bar, tag):
    dtype, got = got.dtype, got.double()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0          # an f16 subnormal's half step
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{tag}: NaN in other places"
    err = torch.where(nan, 0.0, (got - want).abs())
    err = torch.where(got == want, 0.0, err)                          # infinities alike
    bar = torch.where(nan, 1.0, bar + tiny)
    worst = torch.where(err == 0, 0.0, err / bar).max().item() if err.numel() else 0.0
    print(f"[prompt] {tag}: worst error / bar {worst:.3f}", flush=True)
    if not worst <= 1.0:
        i = torch.where(err == 0, 0.0, err / bar).argmax()
        raise AssertionError(f"{tag}: {worst} at {int(i)}: {got.reshape(-1)[i].item()} for {want.reshape(-1)[i].item()}, "
                             f"bar {bar.reshape(-1)[i].item()}")


SHAPES = [
    # lengths, rows behind the last, Hq, Hkv, D, dtype, causal
    ([1], 0, 1, 1, 128, "bf16", True),
    ([64], 0, 4, 1, 128, "bf16", True),
    ([200], 3, 8, 2, 128, "bf16", True),
    ([50] * 7, 0, 6, 3, 128, "f16", True),
    ([0, 33, 0, 1, 129, 128, 0], 40, 4, 2, 128, "bf16", True),
    ([257, 127, 63, 65], 0, 4, 4, 128, "f16", False),
    ([700], 0, 5, 1, 64, "bf16", True),
    ([31, 300, 2], 130, 8, 8, 64, "f16", True),
    ([190, 191], 0, 2, 1, 64, "bf16", False),
    ([513, 40], 0, 6, 2, 32, "f16", True),
    ([97] * 5, 7, 16, 4, 32, "bf16", False),
    ([1] * 200, 0, 2, 1, 32, "bf16", True),
    ([], 5, 2, 1, 64, "bf16", True),
    ([1030], 0, 2, 2, 128, "f16", False),
    # long and few: the forward's waves split the keys
    ([1100], 3, 4, 1, 64, "bf16", True),
    ([1025, 1089], 0, 3, 1, 32, "f16", True),
    ([1345], 0, 8, 2, 128, "bf16", True),
]


@gpu
@pytest.mark.parametrize("lengths,extra,Hq,Hkv,D,dtype,causal", SHAPES)
def test_outputs_and_gradients(device, lengths, extra, Hq, Hkv, D, dtype, causal):
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu(lengths, extra)
    q, k, v, do = (t.to(device) for t in _inputs(N, Hq, Hkv, D, dtype, 900 + N + D))
    if extra:                                       # what lies behind the last sequence is not looked at
        for t in (q, k, v, do):
            t[N - extra:] = float("nan")
    scale = 1 / math.sqrt(D)
    want = _want(q, k, v, cu, causal, scale, do)
    print(f"[prompt] {lengths[:8]} +{extra} {Hq}/{Hkv} D{D} {dtype} causal={causal}", flush=True)
    plain, plse = prompt_attention(q, k, v, cu.to(device), causal=causal, return_lse=True)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = prompt_attention(*leaves, cu.to(device), causal=causal, return_lse=True)
    # the forward of a gradient adds terms below the probabilities' rounding
    assert torch.equal(lse, plse)
    _close(plain, *want["o"], "out alone")
    _close(o.detach(), *want["o"], "out")
    live = torch.isfinite(want["lse"])
    assert torch.equal(torch.isfinite(lse), live)
    assert bool(((lse.double() - want["lse"])[live].abs() < 2e-5).all())
    grads = torch.autograd.grad(o, leaves, do)
    again = torch.autograd.grad(prompt_attention(*leaves, cu.to(device), causal=causal), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "not the same on a second run"
    for n, g in zip(("dq", "dk", "dv"), grads):
        _close(g, *want[n], n)


@gpu
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 3.0])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 32)])
def test_scales(device, scale, dtype, D):
    """Negative, zero and sharp scores."""
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([150, 5])
    q, k, v, do = (t.to(device) for t in _inputs(N, 4, 2, D, dtype, 41))
    want = _want(q, k, v, cu, True, scale, do)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = prompt_attention(*leaves, cu, scale=scale)
    _close(o.detach(), *want["o"], f"scale {scale} out")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
        _close(g, *want[n], f"scale {scale} {n}")


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gain", [2.0 ** -12, 2.0 ** 9])
def test_small_and_large_gradients(device, dtype, gain):
    """Gradients far from one: f16's range is not left and its subnormals cost nothing."""
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([260, 70])
    q, k, v, do = (t.to(device) for t in _inputs(N, 4, 1, 64, dtype, 43))
    do = do * gain
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(prompt_attention(*leaves, cu), leaves, do)
    want = _want(q.detach(), k.detach(), v.detach(), cu, True, 0.125, do)
    for n, g in zip(("dq", "dk", "dv"), grads):
        _close(g, *want[n], f"gain {gain} {n}")


@gpu
def test_growing_scores(device):
    """Each key's score above the last by a few powers of two: the running
    maximum moves in every tile, the sums are rescaled, and slack is used."""
    from omnistack_rs.attention import prompt_attention
    for step in (0.05, 0.7, -0.5):
        N, D = 300, 128
        q = torch.ones(N, 2, D, device=device, dtype=torch.bfloat16)
        k = (torch.arange(N, device=device)[:, None, None] * step / D).to(torch.bfloat16).expand(N, 1, D).contiguous()
        _, _, v, do = (t.to(device) for t in _inputs(N, 2, 1, D, "bf16", 44))
        cu = torch.tensor([0, N])
        want = _want(q, k, v, cu, True, 1.0, do)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        o = prompt_attention(*leaves, cu, scale=1.0)
        _close(o.detach(), *want["o"], f"step {step}")
        for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
            _close(g, *want[n], f"step {step} {n}")


@gpu
def test_layouts_and_out(device):
    """Slices of a fused projection, head-major storage, odd starts: the same
    bits; `out` keeps the rows behind the last sequence."""
    from omnistack_rs.attention import prompt_attention
    lengths, Hq, Hkv, D = [130, 70], 4, 2, 64
    cu, N = _cu(lengths, 9)
    q, k, v, _ = (t.to(device) for t in _inputs(N, Hq, Hkv, D, "bf16", 45))
    cu = cu.to(device)
    want = prompt_attention(q, k, v, cu)
    assert bool((want[200:] == 0).all())
    buf = torch.cat([t.reshape(N, -1) for t in (q, k, v)], 1)
    qs, ks, vs = (t.view(N, -1, D) for t in buf.split([Hq * D, Hkv * D, Hkv * D], 1))
    assert torch.equal(prompt_attention(qs, ks, vs, cu), want)
    hm = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*hm, cu), want)
    odd = [torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*odd, cu), want)
    assert torch.equal(prompt_attention(q, k, v, [0, 130, 200]), want)
    out = torch.full((N, Hq, D), 7.0, device=device, dtype=q.dtype)
    assert prompt_attention(q, k, v, cu, out=out) is out
    assert torch.equal(out[:200], want[:200]) and bool((out[200:] == 7).all())
    torch.full((Hq, N), 3.0, device=device)          # what a fresh lse would hold
    lse = prompt_attention(q, k, v, cu, out=out, return_lse=True)[1]
    assert torch.equal(lse, prompt_attention(q, k, v, cu, return_lse=True)[1]) and bool((lse[:, 200:] == -math.inf).all())
    with pytest.raises(ValueError, match="overlap"):
        prompt_attention(q, k, v, cu, out=q)
    with pytest.raises(ValueError, match="nor itself"):
        prompt_attention(q, k, v, cu, out=torch.empty((N + Hq) * D, device=device, dtype=q.dtype).as_strided((N, Hq, D), (D, D, 1)))
    with pytest.raises(ValueError, match="gradient"):
        prompt_attention(q.clone().requires_grad_(), k, v, cu, out=out)
    with pytest.raises(ValueError, match="gradient"):
        prompt_attention(q, k, v, cu, out=torch.empty_like(q, requires_grad=True))
    with pytest.raises(ValueError, match="rise"):
        prompt_attention(q, k, v, torch.tensor([0, 5, 4], device=device))


@gpu
def test_broadcast_inputs_and_gradients(device):
    """One kv head and one query row spread over many, an output gradient of
    one value: the bits of their copies, and gradients summed over the spread."""
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([70, 140])
    q, k, v, do = (t.to(device) for t in _inputs(N, 4, 1, 64, "bf16", 47))
    cu, q, do = cu.to(device), q[:1], do[:1, :1, :1]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    wide = [t.expand(N, h, 64) for t, h in zip(leaves, (4, 2, 2))]
    o = prompt_attention(*wide, cu)
    grads = torch.autograd.grad(o, wide, do.expand(N, 4, 64), retain_graph=True)
    copies = [t.detach().contiguous().requires_grad_() for t in wide]
    want = prompt_attention(*copies, cu)
    assert torch.equal(o.detach(), want.detach())
    ref = torch.autograd.grad(want, copies, do.expand(N, 4, 64).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(grads, ref))
    sums = torch.autograd.grad(o, leaves, do.expand(N, 4, 64))
    for got, r, d in zip(sums, ref, (0, 1, 1)):
        assert got.shape[d] == 1 and torch.equal(got, r.sum(d, keepdim=True))


@gpu
def test_two_streams_at_once(device):
    """Passes on two streams, queued together, give what each gives alone."""
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([300, 1500])
    cu = cu.to(device)
    sets = [[t.to(device) for t in _inputs(N, 4, 2, 64, "f16", s)] for s in (48, 49)]

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = prompt_attention(*leaves, cu, validate=False)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@gpu
def test_infinity_in_the_last_token_without_a_mask(device):
    """Rows behind a sequence that does not fill its tile have no part in it:
    an infinite value of the last token makes infinite outputs, not NaN, and an
    infinite gradient an infinite dv."""
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([70])
    q, k, v, do = (t.to(device) for t in _inputs(N, 2, 1, 64, "bf16", 47))
    v[69, 0, 3] = float("inf")
    o = prompt_attention(q, k, v, cu, causal=False)
    assert bool((o[:, :, 3] == float("inf")).all()) and bool(torch.isfinite(o[:, :, :3]).all())
    v[69, 0, 3] = 1.0
    do[69, 1, 5] = float("-inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dv = torch.autograd.grad(prompt_attention(*leaves, cu, causal=False), leaves, do)[2]
    assert bool((dv[:, 0, 5] == float("-inf")).all()) and bool(torch.isfinite(dv[:, 0, 6:]).all())


@gpu
def test_far_offsets(device):
    """Token strides of 2 MB: the last tokens lie past 2^32 bytes."""
    from omnistack_rs.attention import prompt_attention
    N, Hq, Hkv, D = 2200, 2, 1, 64
    cu = torch.tensor([0, 100, 2100, N], dtype=torch.int32, device=device)
    q, k, v, do = (t.to(device) for t in _inputs(N, Hq, Hkv, D, "bf16", 48))
    want = prompt_attention(q, k, v, cu)
    buf = torch.empty(N, 1 << 20, dtype=torch.bfloat16, device=device)
    at = 0
    far = []
    for t in (q, k, v, do):
        w = t.shape[1] * D
        buf[:, at:at + w] = t.reshape(N, w)
        far.append(buf[:, at:at + w].view(N, -1, D))
        at += w
    out = buf[:, at:at + Hq * D].view(N, Hq, D)
    assert torch.equal(prompt_attention(*far[:3], cu, out=out), want)
    near = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(prompt_attention(*near, cu), near, do)
    leaves = [t.detach().requires_grad_() for t in far[:3]]
    for a, b in zip(torch.autograd.grad(prompt_attention(*leaves, cu), leaves, far[3]), grads):
        assert torch.equal(a, b)


@gpu
def test_many_short_sequences(device):
    """5000 sequences of 0 to 3 tokens: more than one step of the search for a block's sequence."""
    from omnistack_rs.attention import prompt_attention
    lengths = torch.randint(0, 4, (5000,), generator=_data.gen(49)).tolist()
    cu, N = _cu(lengths, 2)
    q, k, v, do = (t.to(device) for t in _inputs(N, 2, 1, 32, "f16", 50))
    seq = torch.repeat_interleave(torch.arange(5000), torch.tensor(lengths)).to(device)
    n = N - 2
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = prompt_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    # the whole pack as one sequence of which a token sees its own sequence's alone
    for h in range(2):
        Q, K, V = q[:n, h].detach().double(), k[:n, 0].detach().double(), v[:n, 0].detach().double()
        see = (seq[:, None] == seq[None]) & torch.ones(n, n, dtype=torch.bool, device=device).tril()
        p = torch.softmax(torch.where(see, Q @ K.T / math.sqrt(32), -math.inf), -1)
        err = (o[:n, h].double() - p @ V).abs()
        assert bool((err <= 2.0 ** -11 * ((p @ V).abs() + 2 * (p @ V.abs())) + 2.0 ** -25).all())
    assert bool((o[n:] == 0).all()) and all(bool((g[n:] == 0).all()) for g in grads)
    assert all(bool(torch.isfinite(g).all()) for g in grads)


@gpu
def test_capture_and_other_stream(device):
    from omnistack_rs.attention import prompt_attention
    cu, N = _cu([90, 1, 200])
    q, k, v, do = (t.to(device) for t in _inputs(N, 4, 2, 128, "f16", 46))
    cu = cu.to(device)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = prompt_attention(*leaves, cu, validate=False)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    alive = prompt_attention(*leaves, cu, validate=False)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            q.mul_(1.25)
            do.mul_(-0.5)
            cu.copy_(torch.tensor([0, 100 + i, 150, 291]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {i}"


def test_refusals():
    """Checked before any device work: on CPU tensors the last check is the device's."""
    from omnistack_rs.attention import prompt_attention
    q, k = torch.zeros(9, 4, 64, dtype=torch.bfloat16), torch.zeros(9, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP"):
        prompt_attention(q, k, k, [0, 9])
    for args, kw in [((q[0], k, k, [0, 9]), {}), ((q, k, k[:8], [0, 9]), {}), ((q[:, :3], k, k, [0, 9]), {}),
                     ((q[..., :48], k[..., :48], k[..., :48], [0, 9]), {}), ((q.float(), k.float(), k.float(), [0, 9]), {}),
                     ((q, k.half(), k, [0, 9]), {}), ((q, k, k, [0, 10]), {}), ((q, k, k, [1, 9]), {}), ((q, k, k, [0, 5, 4]), {}),
                     ((q, k, k, []), {}), ((q, k, k, [0.0, 9.0]), {}), ((q, k, k, [0, 9]), dict(scale=float("nan"))),
                     ((q, k, k, [0, 9]), dict(scale=float("inf"))), ((q, k, k, [[0, 9]]), {})]:
        with pytest.raises(ValueError):
            prompt_attention(*args, **kw)


def test_native_refusals():
    import ctypes
    from omnistack_rs import _lib
    L = _lib.lib()
    s, odd, far = ((ctypes.c_int64 * 2)(*x) for x in ((128, 64), (127, 64), (1 << 24, 64)))

    def call(q=4096, qs=s, dtype=2, N=5, Hq=2, Hkv=1, D=64, cu=4096, B=1, scale=1.0):
        return L.omni_prompt_attn(q, qs, 4096, s, 4096, s, dtype, N, Hq, Hkv, D, cu, B, scale, 1, 1, 4096, s, None, None, None, None)
    for kw, msg in ((dict(dtype=0), "f16 or bf16"), (dict(D=48), "head_dim"), (dict(Hq=3, Hkv=2), "multiple"), (dict(N=-1), "shape"),
                    (dict(N=1 << 31), "large"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
                    (dict(q=None), "NULL"), (dict(q=4104), "16 bytes"), (dict(qs=odd), "16 bytes"), (dict(qs=far), "stride"),
                    (dict(cu=None), "NULL")):
        assert call(**kw) == _lib.OMNI_EINVAL and msg in _lib.last_error(), (kw, _lib.last_error())
    assert call(N=0, q=None) == 0
    size = L.omni_prompt_attn_backward_workspace_size
    assert size(10, 2, 2, 64, 1) == 10 * 2 * 8 + 4096            # the rows' statistics and the f16 peaks
    assert size(10, 4, 1, 64, 1) in (10 * 4 * 8 + 4096, 10 * 4 * 8 + 4096 + 4 * 2 * 10 * 64 * 4)   # and parts of a group's heads
    assert size(0, 4, 1, 64, 1) == 0 and size(10, 3, 2, 64, 1) == 0
    a = (4096, s)
    rc = L.omni_prompt_attn_backward(*a, *a, *a, 2, 5, 2, 1, 64, 4096, 1, 1.0, 1, *a, *a, 4096, *a, *a, *a, *a, 4096, 100, None)
    assert rc == _lib.OMNI_EWORKSPACE and "workspace" in _lib.last_error()


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D,dtype,G,more", [(128, "bf16", 4, 0), (64, "f16", 1, 0), (32, "bf16", 3, 0), (64, "bf16", 2, 3000)])
def test_infinities_and_nan_stay_with_who_sees_them(device, bad, D, dtype, G, more):
    """A token that holds an infinity or a NaN in q, k, v or the output's
    gradient: what does not see it is as if it held an ordinary number (the
    bars of two computations of one result), other sequences and heads are the
    same bits (f16: the scale of ds may be another power of two, within the
    bars); what sees a NaN is NaN."""
    from omnistack_rs.attention import prompt_attention
    lengths, Hkv = [70, 230, 40 + more], 2           # more: the forward's waves split the keys
    cu, N = _cu(lengths)
    base = [t.to(device) for t in _inputs(N, Hkv * G, Hkv, D, dtype, 60)]
    a, b = 70, 300                                   # the second sequence's tokens

    def run(q, k, v, do):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = prompt_attention(*leaves, cu)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = _want(*base[:3], cu, True, 1 / math.sqrt(D), base[3])
    bars = [2 * want[n][1] for n in ("o", "dq", "dk", "dv")]
    clean = run(*base)
    for at in (0, 1, 33, 63, 64, 100, 229):
        for which in range(4):
            x = [t.clone() for t in base]
            x[which][a + at, 0, 5] = bad             # head 0 (of kv head 0, query head 0)
            got = run(*x)
            for i, (g, c, bar) in enumerate(zip(got, clean, bars)):
                name = f"{'q k v do'.split()[which]} at {at}: {'o dq dk dv'.split()[i]}"
                heads = g.shape[1] // Hkv            # of kv head 0; the other's are untouched
                if dtype == "bf16" or i == 0:
                    assert torch.equal(g[:a], c[:a]) and torch.equal(g[b:], c[b:]), name
                    assert torch.equal(g[a:b, heads:], c[a:b, heads:]), name
                others = [(g[:a].double() - c[:a].double()).abs() <= bar[:a] + 2.0 ** -24,
                          (g[b:].double() - c[b:].double()).abs() <= bar[b:] + 2.0 ** -24]
                assert all(bool(x.all()) for x in others), name
                rows = torch.ones(b - a, g.shape[1], dtype=torch.bool, device=device)     # who may differ
                rows[:, heads:] = False
                if which in (0, 3) and i < 2:        # q, do: query head 0's row alone (do: not the output)
                    rows[:] = False
                    rows[at, 0] = not (which == 3 and i == 0)
                elif which in (0, 3):                # keys that the row sees
                    rows[at + 1:] = False
                elif i < 2:                          # k, v: rows that see the key
                    rows[:at] = False
                elif which == 2 and i == 3:          # v is not in dv
                    rows[:] = False
                same = ~rows
                err = (g[a:b].double() - c[a:b].double()).abs()[same]
                ok = bool((err <= bars[i][a:b][same] + 2.0 ** -24).all())     # NaN fails
                assert ok, f"{name}: {err.max().item()}"
                if math.isnan(bad) and rows.any() and not (which == 3 and i == 1):
                    assert bool(torch.isnan(g[a:b][rows]).any(-1).all()), f"{name}: NaN was lost"


@gpu
@pytest.mark.parametrize("D,dtype,G", [(128, "bf16", 1), (64, "f16", 2), (32, "bf16", 4)])
@pytest.mark.parametrize("at", [5, 40])
def test_rows_without_a_result_leave_the_keys_behind_them_alone(device, at, D, dtype, G):
    """A key with an infinity makes six rows NaN and has no weight in the later
    ones (their scores with it are -inf).  The gradients of the keys behind
    those six rows, which these do not see, are those of the sequence without
    that token."""
    from omnistack_rs.attention import prompt_attention
    n = 150
    q, k, v, do = (t.to(device) for t in _inputs(n, 2 * G, 2, D, dtype, 71))
    k[at, :, 3] = float("inf")
    q[at:, :, 3] = -1.0
    q[at:at + 6, :, 3] = 1.0
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = prompt_attention(*leaves, [0, n])
    _, dk, dv = torch.autograd.grad(o, leaves, do)
    rest = torch.cat([torch.arange(at), torch.arange(at + 1, n)]).to(device)
    want = _want(q[rest], k[rest], v[rest], torch.tensor([0, n - 1]), True, 1 / math.sqrt(D), do[rest])
    assert bool(torch.isnan(o[at:at + 6]).all()) and bool(torch.isnan(dv[at + 1:at + 6]).all())
    for name, got in (("o", o.detach()), ("dk", dk), ("dv", dv)):
        a, b = (t[at + 5:] for t in want[name])
        _close(got[at + 6:], a, b, f"{name} behind the rows")


def test_forward_mode_is_refused():
    """A dual tensor wants a derivative that the kernels do not form: refused
    before any device work, with and without gradients."""
    from torch.autograd import forward_ad
    from omnistack_rs.attention import prompt_attention
    from omnistack_rs.attention.prompt import _PromptAttention
    q, k = torch.zeros(9, 4, 64, dtype=torch.bfloat16), torch.zeros(9, 2, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        for i in range(3):
            for grad in (False, True):
                args = [q, k, k]
                args[i] = forward_ad.make_dual(args[i].clone().requires_grad_(grad), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    prompt_attention(*args, [0, 9])
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    prompt_attention(*args, [0, 9])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            prompt_attention(q, k, k, [0, 9], out=forward_ad.make_dual(q.clone(), torch.ones_like(q)))
        with pytest.raises(RuntimeError, match="HIP"):
            prompt_attention(q, k, k, [0, 9])
        dual = forward_ad.make_dual(q.clone(), torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="gradient has no forward-mode"):      # a tangent of the gradient
            _PromptAttention.backward(None, dual, None)


def test_scales_that_leave_fp32_are_refused():
    """The kernels multiply the scale by log2 e: 2.35e38 is the last that stays
    finite there; the refusal starts at 2.3e38."""
    import ctypes
    from omnistack_rs import _lib
    from omnistack_rs.attention import prompt_attention
    q, k = torch.zeros(9, 4, 64, dtype=torch.bfloat16), torch.zeros(9, 2, 64, dtype=torch.bfloat16)
    s = (ctypes.c_int64 * 2)(128, 64)
    for x in (2.4e38, -2.4e38, 2.9e38):
        with pytest.raises(ValueError, match="scale"):
            prompt_attention(q, k, k, [0, 9], scale=x)
        rc = _lib.lib().omni_prompt_attn(4096, s, 4096, s, 4096, s, 2, 0, 2, 1, 64, 4096, 1, x, 1, 1, 4096, s, None, None, None, None)
        assert rc == _lib.OMNI_EINVAL and "scale" in _lib.last_error()
    assert math.isfinite(torch.tensor(2.3e38 * 1.44269504, dtype=torch.float32).item())
    with pytest.raises(RuntimeError, match="HIP"):
        prompt_attention(q, k, k, [0, 9], scale=-2.3e38)
    assert _lib.lib().omni_prompt_attn(4096, s, 4096, s, 4096, s, 2, 0, 2, 1, 64, 4096, 1, 2.29e38, 1, 1, 4096, s, None, None, None, None) == 0


# What rounding the output left.  For a gradient the forward stores it, out_rest,
# and takes the first 64 keys' probabilities as two 16-bit numbers each, p and
# what rounding p left, off by u^2 p together.  With e2 = u^2 + 2 X + 2^-20 (the
# probability's own errors, as at the top) weights that sum to one leave
# e2 sum_s p |v - o|; two fp32 sums over at most 64 keys, two products each, leave
# 128 u32 (sum_s p |v| + |o|); out_rest is rounded, u^2 |o| (f16: or half a
# subnormal step, and the remainders of p half a step 2^-32 of the largest p).

def _with_rest(q, k, v, lengths, scale, do):
    """64-bit results of causal sequences of at most 64 tokens: o, dq, dk with
    bars that grant delta what o + out_rest is off by and nothing for a rounded o;
    and what o alone in place of o + out_rest does to dq and dk."""
    u, D, G, f16 = torch.finfo(q.dtype).eps / 2, q.shape[2], q.shape[1] // k.shape[1], q.dtype == torch.float16
    q64, k64, v64, g64 = (t.double() for t in (q, k, v, do))
    res = {n: [torch.zeros_like(t) for _ in range(3)] for n, t in (("o", q64), ("dq", q64), ("dk", k64))}
    sub = 2.0 ** -25 if f16 else 0.0
    least = 2.0 ** -38 * 2 * g64.norm(dim=-1).max() * v64.norm(dim=-1).max() if f16 else 2.0 ** -126
    a = 0
    for n in lengths:
        see = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(q.shape[1]):
            Q, K, V, g = q64[a:a + n, h], k64[a:a + n, h // G], v64[a:a + n, h // G], g64[a:a + n, h]
            p = torch.softmax(torch.where(see, Q @ K.T * scale, -math.inf), -1)
            X = ((D + 2) * U32 * abs(scale) * (Q.abs() @ K.abs().T) * see).amax(-1, keepdim=True)
            O = p @ V
            e2 = u * u + 2 * X + 2.0 ** -20
            spread = (p[:, :, None] * (V[None] - O[:, None]).abs()).sum(1)
            ob = e2 * spread + 128 * U32 * (p @ V.abs() + O.abs()) + u * u * O.abs() + sub
            if f16:
                ob = ob + 2.0 ** -32 * ((see.double() @ V.abs()) + see.sum(-1, keepdim=True) * O.abs())
            dp, delta = g @ V.T, (g * O).sum(-1, keepdim=True)
            Y = D * U32 * (g.abs() @ V.abs().T + (g.abs() * O.abs()).sum(-1, keepdim=True)) + (g.abs() * ob).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            dsb = p * Y + (2 * u + 2 * X + 2.0 ** -20) * ds.abs() + least * see
            off = p * (g * (O.to(q.dtype).double() - O)).sum(-1, keepdim=True)       # of ds, from a rounded o
            res["o"][0][a:a + n, h], res["o"][1][a:a + n, h] = O, ob
            for name, hh, x, b, f in (("dq", h, ds @ K, dsb @ K.abs(), off @ K), ("dk", h // G, ds.T @ Q, dsb.T @ Q.abs(), off.T @ Q)):
                for r, y in zip(res[name], (x * scale, b * abs(scale), f * scale)):
                    r[a:a + n, hh] += y
        a += n
    for name in ("dq", "dk"):
        res[name][1] += u * res[name][0].abs()
    return res


REST = [("bf16", 128, 4, 2), ("bf16", 64, 3, 1), ("f16", 32, 4, 4)]


def _rest_inputs(D, dtype, Hq, Hkv, seed):
    """v within half of 8, in sixteenths: dp - delta is a small difference of large terms."""
    lengths = [64, 1, 17, 40, 2]
    q, k, v, do = _inputs(sum(lengths), Hq, Hkv, D, dtype, seed, 0.25)
    return lengths, q, k, (8 + (v.float().clamp(-2, 2) * 4).round() / 16).to(DT[dtype]), do


@pytest.mark.parametrize("dtype,D,Hq,Hkv", REST)
def test_the_rests_bars_would_notice(dtype, D, Hq, Hkv):
    """A gradient from o alone, or with out_rest's sign turned (twice as far off), leaves the bars."""
    lengths, q, k, v, do = _rest_inputs(D, dtype, Hq, Hkv, 91)
    res = _with_rest(q, k, v, lengths, 1 / math.sqrt(D), do)
    for name in ("dq", "dk"):
        x, bar, off = res[name]
        assert (off.abs() / bar).max() > 2, name
    O, bar, _ = res["o"]
    assert ((O.to(DT[dtype]).double() - O).abs() / bar).max() > 2
    # probabilities without their remainders, on values around 0
    q, k, v, _ = _inputs(64, Hq, Hkv, D, dtype, 92)
    res = _with_rest(q, k, v, [64], 1 / math.sqrt(D), torch.zeros_like(q))
    p = torch.exp(torch.where(torch.ones(64, 64).tril() > 0, q[:, 0].double() @ k[:, 0].double().T / math.sqrt(D), -math.inf))
    p = (p / p.amax(-1, keepdim=True)).to(DT[dtype]).double()
    o = (p / p.sum(-1, keepdim=True)) @ v[:, 0].double()
    assert ((o - res["o"][0][:, 0]).abs() / res["o"][1][:, 0]).max() > 2


@gpu
@pytest.mark.parametrize("dtype,D,Hq,Hkv", REST)
def test_out_and_its_rest(device, dtype, D, Hq, Hkv):
    """out + out_rest is the 64-bit output, and delta is taken from both: dq and
    dk of values that lie close together."""
    from omnistack_rs.attention import prompt, prompt_attention
    lengths, *near = _rest_inputs(D, dtype, Hq, Hkv, 91)
    for which, (q, k, v, do) in (("near", near), ("around 0", _inputs(sum(lengths), Hq, Hkv, D, dtype, 92))):
        q, k, v, do = (t.to(device) for t in (q, k, v, do))
        cu = _cu(lengths)[0].to(device)
        want = _with_rest(q, k, v, lengths, 1 / math.sqrt(D), do)
        o, _, rest = prompt._forward(q, k, v, cu, 1 / math.sqrt(D), True, None, True, device, True)
        assert bool((rest != 0).any())
        _close(o.double() + rest.double(), *want["o"][:2], f"{which}: out and rest")
        leaves = [t.requires_grad_() for t in (q, k, v)]
        grads = torch.autograd.grad(prompt_attention(*leaves, cu), leaves, do)
        _close(grads[0], *want["dq"][:2], f"{which}: dq")
        _close(grads[1], *want["dk"][:2], f"{which}: dk")
