"""What stands between a model's projections and the packed cache: the norm and
position rotation of query and key heads, and the attention of whole prompts
packed one after another, each with its gradient.

A case is a dict of plain values:

    op          qk_norm_rope, the norm of every query and key head and the
                rotation by position in one pass, or
                prompt_attention, softmax attention within each sequence of a
                packed batch, grouped heads
    direction   forward, or train: the outputs and every gradient for a given
                gradient of the outputs
    dtype       of q, k, v (f32, f16, bf16)
    Hq, Hkv, D  query heads, key/value heads, head_dim
    tokens, axes, rotary, norm, pairs, layout, first
                (qk_norm_rope) rows; position axes (1 text, 3 time x height x
                width); dims that turn; whether heads are normed; halves or
                neighbours as pairs; heads of their own or slices of one fused
                projection; the position that the rows start from
    lengths, causal
                (prompt_attention) the packed sequences' lengths, as text

`listed` has the sizes of the benchmark's configurations (64 users of 50
tokens or of one new token, 8 chunks of 512 tokens, 32 query heads over 8,
head_dim 128 and the pruned 32) and prompts up to 32768 tokens; `draw` spreads
the same kinds over their ranges.
"""
from __future__ import annotations

import math
import os
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omnistack-rs_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 10000.0


def _rope(name, **kw):
    c = dict(op="qk_norm_rope", direction="forward", dtype="bf16", Hq=32, Hkv=8, D=128, tokens=64, axes=1, rotary=128,
             norm=True, pairs="halves", layout="heads", first=0)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _prompt(name, **kw):
    c = dict(op="prompt_attention", direction="forward", dtype="bf16", Hq=32, Hkv=8, D=128, lengths="50", causal=True)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _text(lengths):
    return ",".join(str(n) for n in lengths)


def listed():
    return [
        # one decode step of 64 users: a token each, far into their histories
        _rope("rope_step_64", tokens=64, first=100000),
        # 8 chunks of 512 prompt tokens, q and k as slices of a fused projection's output
        _rope("rope_chunks_8x512", tokens=4096, layout="fused"),
        # a video clip's patches: time, height and width, an odd number of them, rotation only
        _rope("rope_video_9001", tokens=9001, dtype="f16", axes=3, Hq=16, Hkv=16, norm=False),
        # the pruned head_dim in f32, as the fidelity checks keep their tensors, neighbouring pairs
        _rope("rope_f32_d32_16391", tokens=16391, dtype="f32", D=32, rotary=32, pairs="neighbours"),
        # a long-context prefill's tokens
        _rope("rope_prompt_65536", tokens=65536, layout="fused"),
        # a training step's tokens: outputs, input gradients and the norms' weight gradients
        _rope("rope_train_8192", tokens=8192, direction="train"),
        # the users of a serving batch, each with its whole history of 50 tokens
        _prompt("prompt_64x50", lengths=_text([50] * 64)),
        # one ordinary prompt
        _prompt("prompt_2048", lengths="2048"),
        # a batch as a scheduler packs it: one token to several thousand
        _prompt("prompt_ragged_f16", dtype="f16", lengths="1,17,130,513,1024,2047,4099,6001"),
        # a long document
        _prompt("prompt_32768", lengths="32768"),
        # adapter training on packed sequences
        _prompt("train_ragged", direction="train", lengths="4096,2000,1333,700,63"),
        # whole histories seen in both directions, pruned head_dim, many short sequences
        _prompt("train_d32_f16", direction="train", dtype="f16", Hq=16, Hkv=4, D=32, causal=False,
                lengths=_text([40 + 37 * i for i in range(24)])),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = rng.choice([(32, 8), (16, 4), (8, 8), (16, 16), (10, 2), (7, 1), (40, 8), (64, 8)])
    if rng.random() < 0.5:
        D = rng.choice([128, 128, 32, 64, 256])
        # 2^26 elements at most, so that a pass moves less than the listed 65536 tokens' does
        most = min(65536, (1 << 26) // (sum(heads) * D))
        direction = rng.choice(["forward", "forward", "train"])
        n = _log_int(rng, 1, most // (2 if direction == "train" else 1))
        return _rope(None, Hq=heads[0], Hkv=heads[1], D=D, tokens=n, direction=direction,
                     dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), axes=rng.choice([1, 1, 2, 3]),
                     rotary=rng.choice([D, D, D // 2]), norm=rng.random() < 0.75,
                     pairs=rng.choice(["halves", "halves", "neighbours"]), layout=rng.choice(["heads", "fused"]),
                     first=rng.choice([0, 0, _log_int(rng, 10, 2000000)]))
    D = rng.choice([128, 128, 32, 64])
    direction = rng.choice(["forward", "forward", "train"])
    causal = rng.random() < 0.75
    total = _log_int(rng, 8, 8192 if direction == "train" else 16384)
    pieces = _log_int(rng, 1, 96)
    cuts = sorted(rng.randint(0, total) for _ in range(pieces - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]      # zeros among them now and then
    return _prompt(None, Hq=heads[0], Hkv=heads[1], D=D, direction=direction, causal=causal,
                   dtype=rng.choice(["bf16", "bf16", "f16"]), lengths=_text(lengths))


# ── inputs ──────────────────────────────────────────────────────────────

def _lengths(case):
    return [int(x) for x in case["lengths"].split(",")]


def _inv_freq(case):
    """float64 frequencies of the R/2 pairs and each pair's axis: thirds (or
    halves) of the pairs in turn, time first."""
    n, A = case["rotary"] // 2, case["axes"]
    f = [BASE ** (-i / n) for i in range(n)]
    cuts = [n * a // A for a in range(A + 1)]
    axis = [a for a in range(A) for _ in range(cuts[a + 1] - cuts[a])]
    return f, axis


def _positions(case, g):
    """int64 (axes, tokens)."""
    N, A, first = case["tokens"], case["axes"], case["first"]
    if A == 1:
        if N <= 256 and first:                      # single tokens of as many users
            return torch.randint(first // 2, first + 1, (1, N), generator=g, device=DEV)
        return (torch.arange(N, device=DEV) + first)[None]
    side = max(1, int(N ** (1.0 / 3.0)))            # a clip of side x side patches a frame
    i = torch.arange(N, device=DEV)
    grid = [i // (side * side) + first, (i // side) % side, i % side]
    return torch.stack(grid[:A])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt, Hq, Hkv, D = DTYPES[case["dtype"]], case["Hq"], case["Hkv"], case["D"]

    def heads(n, h):
        # projections' rows: heads of different strength, unit variance on average
        gain = 0.5 + torch.rand(h, 1, generator=g, device=DEV)
        return (torch.randn(n, h, D, generator=g, device=DEV) * gain).to(dt)

    s = dict(case=case)
    if case["op"] == "qk_norm_rope":
        N = case["tokens"]
        if case["layout"] == "fused":
            s["qkv"] = heads(N, Hq + 2 * Hkv).reshape(N, (Hq + 2 * Hkv) * D)
        else:
            s["q"], s["k"] = heads(N, Hq), heads(N, Hkv)
        s["positions"] = _positions(case, g)
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"], s["wk"] = (1 + 0.2 * torch.randn(2, D, generator=g, device=DEV)).to(dt)
        if case["direction"] == "train":
            s["dq"], s["dk"] = heads(N, Hq), heads(N, Hkv)
        f, axis = _inv_freq(case)
        s["freq"] = torch.tensor(f, dtype=torch.float64, device=DEV)
        s["axis"] = torch.tensor(axis, device=DEV)
        if own:
            from omnistack_rs.kernels.rope import RotaryEmbedding
            s["rotary"] = RotaryEmbedding(D, rotary_dim=case["rotary"], inv_freq=f, pair_axes=axis,
                                          interleaved=case["pairs"] == "neighbours", device=DEV)
        return s
    L = _lengths(case)
    N = sum(L)
    s["lengths"] = L
    s["q"], s["k"], s["v"] = heads(N, Hq), heads(N, Hkv), heads(N, Hkv)
    s["cu_seqlens"] = torch.tensor([sum(L[:i]) for i in range(len(L) + 1)], dtype=torch.int32, device=DEV)
    if case["direction"] == "train":
        s["do"] = heads(N, Hq)
    return s


def _qk(s):
    """q (N, Hq, D) and k (N, Hkv, D) as the program has them."""
    if "q" in s:
        return s["q"], s["k"]
    c = s["case"]
    n, a, b = c["tokens"], c["Hq"] * c["D"], (c["Hq"] + c["Hkv"]) * c["D"]
    return s["qkv"][:, :a].view(n, c["Hq"], c["D"]), s["qkv"][:, a:b].view(n, c["Hkv"], c["D"])


# ── one pass ────────────────────────────────────────────────────────────

def run(s):
    c = s["case"]
    if own:
        return (_own_rope if c["op"] == "qk_norm_rope" else _own_prompt)(s)
    return (_plain_rope if c["op"] == "qk_norm_rope" else _plain_prompt)(s)


def _own_rope(s):
    from omnistack_rs.kernels.rope import qk_norm_rope
    q, k = _qk(s)
    if s["case"]["direction"] == "forward":
        return qk_norm_rope(q, k, s["positions"], s["rotary"], s["wq"], s["wk"], EPS)
    leaves = [q.detach().requires_grad_(), k.detach().requires_grad_()]
    if s["wq"] is not None:
        leaves += [s["wq"].detach().requires_grad_(), s["wk"].detach().requires_grad_()]
    y = qk_norm_rope(leaves[0], leaves[1], s["positions"], s["rotary"], *(leaves[2:] or (None, None)), EPS)
    grads = torch.autograd.grad(y, leaves, (s["dq"], s["dk"]))
    return (*(t.detach() for t in y), *grads)


def _own_prompt(s):
    from omnistack_rs.attention import prompt_attention
    c = s["case"]
    if c["direction"] == "forward":
        return prompt_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], causal=c["causal"], validate=False)
    leaves = [s[x].detach().requires_grad_() for x in ("q", "k", "v")]
    o = prompt_attention(*leaves, s["cu_seqlens"], causal=c["causal"], validate=False)
    return (o.detach(), *torch.autograd.grad(o, leaves, s["do"]))


def _turn(x, cos, sin, pairs):
    """Rotate the first 2 * cos.shape[-1] dims of x (N, H, D), the rest as is."""
    R = 2 * cos.shape[-1]
    out = x.clone()
    if pairs == "halves":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_rope(s):
    c = s["case"]
    theta = s["positions"][s["axis"]].double().T * s["freq"]          # (N, R/2), far positions
    cos, sin = theta.cos().float()[:, None], theta.sin().float()[:, None]
    q, k = _qk(s)
    train = c["direction"] == "train"
    outs, dxs, dws = [], [], []
    for x, w, dy in ((q, s["wq"], s.get("dq")), (k, s["wk"], s.get("dk"))):
        dt, x = x.dtype, x.float()
        if w is not None:
            w = w.float()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            z = x * r * w
        else:
            z = x
        outs.append(_turn(z, cos, sin, c["pairs"]).to(dt))
        if not train:
            continue
        dz = _turn(dy.float(), cos, -sin, c["pairs"])
        if w is None:
            dxs.append(dz.to(dt))
            continue
        gxr = dz * x * r
        dws.append(gxr.double().sum((0, 1)).to(dt))                   # a long sum
        dxs.append((r * (dz * w - x * r * (gxr * w).mean(-1, keepdim=True))).to(dt))
    return (*outs, *dxs, *dws)


_ROWS = 4096             # query rows whose scores are held at once,
_SCORES = 1 << 30        # and scores


def _plain_prompt(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    N, Hq, D = q.shape
    Hkv = k.shape[1]
    G, scale, dt = Hq // Hkv, 1.0 / math.sqrt(D), q.dtype
    train = c["direction"] == "train"
    out = torch.empty_like(q)
    if train:
        dq = torch.empty_like(q)
        dk, dv = torch.empty_like(k), torch.empty_like(v)

    def grouped(x):                                                   # (n, m * G, D) -> (m, G * n, D)
        n = x.shape[0]
        return x.float().view(n, -1, G, D).permute(1, 2, 0, 3).reshape(-1, G * n, D)

    def ungrouped(x, n):
        return x.view(-1, G, n, D).permute(2, 0, 1, 3).reshape(n, -1, D).to(dt)

    at = 0
    for L in s["lengths"]:
        step = max(1, min(Hkv, _SCORES // max(1, G * min(L, _ROWS) * L)))   # kv heads at once
        for h in range(0, Hkv if L else 0, step):
            ks = slice(h, h + step)
            hs = slice(h * G, min(h + step, Hkv) * G)
            kf = k[at:at + L, ks].float().transpose(0, 1).contiguous()
            vf = v[at:at + L, ks].float().transpose(0, 1).contiguous()
            if train:
                dkf, dvf = torch.zeros_like(kf), torch.zeros_like(vf)
            for t0 in range(0, L, _ROWS):
                n = min(_ROWS, L - t0)
                S = t0 + n if c["causal"] else L                      # keys that a row here can see
                rows = slice(at + t0, at + t0 + n)
                qf = grouped(q[rows, hs])
                x = qf @ kf[:, :S].transpose(1, 2) * scale
                if c["causal"]:
                    t = torch.arange(t0, t0 + n, device=DEV)
                    x.view(-1, G, n, S).masked_fill_(t[:, None] < torch.arange(S, device=DEV), float("-inf"))
                x = torch.exp(x - x.amax(-1, keepdim=True))
                p = x.div_(x.sum(-1, keepdim=True))
                o = p @ vf[:, :S]
                out[rows, hs] = ungrouped(o, n)
                if train:
                    do = grouped(s["do"][rows, hs])
                    ds = do @ vf[:, :S].transpose(1, 2)
                    ds = p * (ds - (do * o).sum(-1, keepdim=True))
                    dq[rows, hs] = ungrouped(ds @ kf[:, :S] * scale, n)
                    dkf[:, :S] += ds.transpose(1, 2) @ qf * scale
                    dvf[:, :S] += p.transpose(1, 2) @ do
            if train:
                dk[at:at + L, ks], dv[at:at + L, ks] = dkf.transpose(0, 1).to(dt), dvf.transpose(0, 1).to(dt)
        at += L
    return (out, dq, dk, dv) if train else out


# ── what a pass cannot do without ───────────────────────────────────────

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    train = case["direction"] == "train"
    if case["op"] == "qk_norm_rope":
        N = case["tokens"]
        el = N * (Hq + Hkv) * D
        w = 2 * D * size if case["norm"] else 0
        # x in, y out; train: dy in, dx and dw out as well
        nbytes = el * size * (4 if train else 2) + 8 * N * case["axes"] + w * (2 if train else 1)
        return {"bytes": nbytes, "flops": el * (7 if case["norm"] else 3) * (3 if train else 1)}
    L = _lengths(case)
    N = sum(L)
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in L) * Hq
    # q, k, v in and o out; train: do in and dq, dk, dv out as well
    el = N * D * (Hq * 2 + Hkv * 2) * (2 if train else 1)
    # q.k and p.v; train: and dp, dv, dk, dq
    return {"bytes": el * size + 4 * (len(L) + 1), "flops": pairs * D * (12 if train else 4)}


# ── the definition in 64 bits ───────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["op"] == "qk_norm_rope" else _exact_prompt(case, s)


def _exact_rope(case, s):
    """Each pair as a complex number: (a + ib) e^{i theta}; the gradient is the
    transposed map applied to dy, and the norm's Jacobian written out."""
    R = case["rotary"]
    theta = s["freq"][None] * s["positions"].double()[s["axis"]].T
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    halves = case["pairs"] == "halves"

    def pairs_of(x):
        t = x[..., :R]
        t = t.unflatten(-1, (2, R // 2)).transpose(-1, -2) if halves else t.unflatten(-1, (R // 2, 2))
        return torch.view_as_complex(t.contiguous())

    def back(zc, x):
        t = torch.view_as_real(zc)
        t = t.transpose(-1, -2) if halves else t
        return torch.cat([t.reshape(*x.shape[:-1], R), x[..., R:]], -1)

    ys, dxs, dws = [], [], []
    for x, w, dy in zip(_qk(s), (s["wq"], s["wk"]), (s.get("dq"), s.get("dk"))):
        x = x.double()
        if w is not None:
            w = w.double()
            rms = torch.sqrt(torch.linalg.vecdot(x, x)[..., None] / x.shape[-1] + EPS)
            xhat = x / rms
            z = xhat * w
        else:
            z = x
        ys.append(back(pairs_of(z) * turn, z))
        if dy is not None:
            dy = dy.double()
            dz = back(pairs_of(dy) * turn.conj(), dy)
            if w is None:
                dxs.append(dz)
            else:
                dws.append(torch.einsum("nhd,nhd->d", dz, xhat))
                u = dz * w
                dxs.append((u - xhat * torch.linalg.vecdot(u, xhat)[..., None] / x.shape[-1]) / rms)
    return (*ys, *dxs, *dws)


def _exact_prompt(case, s):
    """Row by row of the definition, in blocks of rows of one query head."""
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    N, Hq, D = q.shape
    G, train = Hq // k.shape[1], case["direction"] == "train"
    o = torch.empty_like(q)
    if train:
        do = s["do"].double()
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for L in s["lengths"]:
        end = start + L
        for h in range(Hq):
            kh = h // G
            for a in range(start, end, 2048):
                b = min(a + 2048, end)
                last = b if case["causal"] else end
                K, V = k[start:last, kh], v[start:last, kh]
                score = q[a:b, h] @ K.T / D ** 0.5
                if case["causal"]:
                    seen = torch.arange(start, last, device=DEV)[None] <= torch.arange(a, b, device=DEV)[:, None]
                    score = torch.where(seen, score, -math.inf)
                P = torch.softmax(score, -1)
                O = P @ V
                o[a:b, h] = O
                if train:
                    g = do[a:b, h]
                    dP = g @ V.T
                    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) / D ** 0.5
                    dq[a:b, h] = dS @ K
                    dk[start:last, kh] += dS.T @ q[a:b, h]
                    dv[start:last, kh] += P.T @ g
        start = end
    return (o, dq, dk, dv) if train else o
