"""The prompt's path from the projections to the packed cache, and a query
adapter trained through it: qk_norm_rope, prompt_attention, PagedKVCache.append
and paged_attention one after another."""
import math

import pytest
import torch

from tests import _data

pytestmark = pytest.mark.gpu


def _rope64(x, w, pos, eps=1e-6):
    """Norm and rotation in 64 bits, halves as pairs, base 10000."""
    D = x.shape[-1]
    z = x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    t = pos.double()[:, None] * torch.tensor([10000.0 ** (-2 * i / D) for i in range(D // 2)], dtype=torch.float64, device=x.device)
    c, s = t.cos()[:, None], t.sin()[:, None]
    a, b = z[..., :D // 2], z[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _attn64(q, k, v, cu):
    G, out = q.shape[1] // k.shape[1], []
    for a, b in zip(cu[:-1], cu[1:]):
        Q, K, V = q[a:b].transpose(0, 1), k[a:b].repeat_interleave(G, 1).transpose(0, 1), v[a:b].repeat_interleave(G, 1).transpose(0, 1)
        s = (Q @ K.transpose(1, 2) / math.sqrt(q.shape[-1])).masked_fill(
            ~torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril(), -math.inf)
        out.append((torch.softmax(s, -1) @ V).transpose(0, 1))
    return torch.cat(out)


def test_prompts_into_pages_and_on(device):
    """Ragged prompts: norm and rotation in place on a fused projection's
    slices, attention, keys and values into pages; then a step of one token a
    sequence.  The attention is that of 64-bit heads within three roundings
    (q and k rounded once each, then the attention's own bar of two for
    weights and output; scores of unit-norm heads of 128 move by 2 u sqrt(128)
    at most, a factor of 1 + 2^-3 on weights at bf16's u = 2^-8, far less in
    the mean); the step is omni_attn's over a contiguous cache of the same keys
    and values, within the paged kernel's bar of 2e-3."""
    from omnistack_rs.attention import prompt_attention
    from omnistack_rs.cache import PagedKVCache, paged_attention
    from omnistack_rs.kernels.fused_attention import omni_attn
    from omnistack_rs.kernels.quantize import PackedKVEncoder
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    lengths, Hq, Hkv, D = [130, 17, 64], 8, 2, 128
    cu = [0, 130, 147, 211]
    N, B = cu[-1], len(lengths)
    g = _data.gen(70)
    qkv = torch.randn(N, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).to(device)
    step = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).to(device)
    wq, wk = ((1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(device) for _ in range(2))
    heads = lambda t: [x.view(t.shape[0], -1, D) for x in t.split([Hq * D, Hkv * D, Hkv * D], 1)]  # noqa: E731
    q, k, v = heads(qkv)
    pos = torch.cat([torch.arange(n) for n in lengths]).to(device)
    want = _attn64(_rope64(q.double(), wq.double(), pos), _rope64(k.double(), wk.double(), pos), v.double(), cu)
    rotary = RotaryEmbedding(D, device=device)
    qk_norm_rope(q, k, pos, rotary, wq, wk, out=(q, k))
    out = prompt_attention(q, k, v, cu)
    err = (out.double() - want).norm() / want.norm()
    print(f"[path] prompt attention off by {err.item():.2e}", flush=True)
    assert err.item() < 3 * 2.0 ** -8

    cb = _data.gaussian_codebook(Hkv).to(device)
    enc = PackedKVEncoder(cb, Hkv, user_id=3, rotate=True, dtype=torch.bfloat16)
    cache = PagedKVCache(64, Hkv, 16, D, device=device)
    pages = [cache.allocate(n + 1) for n in lengths]
    table = cache.page_table(pages)
    bhtd = lambda t: t.transpose(0, 1)[None].contiguous()  # noqa: E731
    for b in range(B):
        cache.append(enc, bhtd(k[cu[b]:cu[b + 1]]), bhtd(v[cu[b]:cu[b + 1]]), table[b:b + 1],
                     torch.zeros(1, dtype=torch.int32, device=device))
    # a token more of each sequence, in the cache's own layout
    sq, sk, sv = (t[:, :, None] for t in heads(step))                       # (B, heads, 1, D)
    at = torch.tensor(lengths, dtype=torch.int32, device=device)
    sq, sk = qk_norm_rope(sq, sk, at[:, None], rotary, wq, wk)
    cache.append(enc, sk, sv.contiguous(), table, at)
    got = paged_attention(sq, cache, table, at + 1, cb, user_id=3, rotate_q=True)
    for b, n in enumerate(lengths):
        K = torch.cat([bhtd(k[cu[b]:cu[b + 1]]), sk[b:b + 1]], 2)
        V = torch.cat([bhtd(v[cu[b]:cu[b + 1]]), sv[b:b + 1]], 2)
        (kn, kq, kr), (vn, _, _) = enc.encode(K, V.contiguous())
        one = omni_attn(sq[b:b + 1], kn, kq, kr, vn, cb, user_id=3, rotate_q=True)
        assert bool((got[b:b + 1] - one).abs().max() < 2e-3), b


def test_query_adapter_gradients(device):
    """d loss / d (A, B) of a low-rank update of the queries, through the norm,
    the rotation and the attention, against 64 bits.  Roundings to bf16 on the
    way: the update's two products, q, the rotated q, the output's gradient
    path (dq of the attention, of the norm, and the two products back): nine,
    each u = 2^-8 of its tensor at most; random matrices carry a relative error
    on about as it is (a factor of 2 is allowed): 18 u."""
    from omnistack_rs.attention import prompt_attention
    from omnistack_rs.kernels.rope import RotaryEmbedding, qk_norm_rope
    cu, Hq, Hkv, D, hidden, rank = [0, 96, 200], 4, 2, 64, 256, 16
    N = cu[-1]
    g = _data.gen(71)
    mk = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.bfloat16).to(device)  # noqa: E731
    x, wq = mk(N, hidden), mk(hidden, Hq * D, scale=hidden ** -0.5)
    k, v, target = mk(N, Hkv, D), mk(N, Hkv, D), mk(N, Hq, D)
    A, Bm = mk(hidden, rank, scale=hidden ** -0.5), mk(rank, Hq * D, scale=rank ** -0.5)
    w = mk(D, scale=0.1) + 1
    pos = torch.cat([torch.arange(96), torch.arange(104)]).to(device)
    rotary = RotaryEmbedding(D, device=device)
    A.requires_grad_()
    Bm.requires_grad_()
    q = (x @ wq + x @ A @ Bm).view(N, Hq, D)
    q, kr = qk_norm_rope(q, k, pos, rotary, w, w)
    grads = torch.autograd.grad(prompt_attention(q, kr, v, cu), (A, Bm), target)
    A64, B64 = (t.detach().double().requires_grad_() for t in (A, Bm))
    x64, w64 = x.double(), w.double()
    q64 = _rope64((x64 @ wq.double() + x64 @ A64 @ B64).view(N, Hq, D), w64, pos)
    o64 = _attn64(q64, _rope64(k.double(), w64, pos), v.double(), cu)
    want = torch.autograd.grad(o64, (A64, B64), target.double())
    for n, a, b in zip("AB", grads, want):
        err = ((a.double() - b).norm() / b.norm()).item()
        print(f"[path] d loss / d {n} off by {err:.2e}", flush=True)
        assert err < 18 * 2.0 ** -8, n
