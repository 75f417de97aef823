"""Serving over the paged compressed cache beyond one token after another: the
attention of a tree of drafted tokens, and attention over the blocks (pages)
that a cheap score selects for each query.

A case is a dict of plain values:

    op          tree, softmax attention of each sequence's drafted tokens over
                its cached tokens and those drafted tokens that the tree lets
                it see, or
                blocks, the selection of each query's blocks by the bounds of
                their keys' codes and softmax attention over the selected ones
    dtype       of q and the output (f16, bf16)
    Hq, Hkv     query heads, key/value heads (head_dim 128)
    B, lo, hi   sequences and their lengths, spread from lo to hi, the
                drafted tokens among them
    page        tokens of a page
    T           query tokens of a sequence
    qjl         whether the keys' residual signs take part
    rotate      whether the call rotates q by the signed Hadamard transform
    ragged      (tree) sequences have from none to T drafted tokens
    top         (blocks) blocks that each query and kv head reads, the first
                one and the one of the query's own token among them

`listed` has the sizes of the benchmark's configurations (64 users of 50
tokens, 32 sequences of 8192, 8 of 16384, 32 query heads over 8) and caches up
to 131072 tokens; `draw` spreads the same kinds over their ranges.
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
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
D = 128
UID = 42
SCALE = 1.0 / math.sqrt(D)
# Max's (1960) 16-level quantizer of N(0, 1)
_LEVELS = (0.1284, 0.3881, 0.6568, 0.9424, 1.2562, 1.6181, 2.0690, 2.7326)


def _tree(name, **kw):
    c = dict(op="tree", dtype="bf16", Hq=32, Hkv=8, B=1, lo=300, hi=300, page=16, T=8, qjl=True, rotate=True, ragged=False)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _blocks(name, **kw):
    c = dict(op="blocks", dtype="bf16", Hq=32, Hkv=8, B=1, lo=8192, hi=8192, page=16, T=1, qjl=True, rotate=True, top=64)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one reader's four guesses after a short prompt
        _tree("tree_1x300_t4", T=4),
        # a serving batch's users, eight guesses each after their 50 tokens
        _tree("tree_64x58_t8", B=64, lo=58, hi=58, T=8),
        # as a scheduler packs it: mixed lengths, every sequence with its own number of guesses, heads of their own
        _tree("tree_48_ragged_f16", B=48, lo=75, hi=2917, T=12, Hq=16, Hkv=16, page=64, dtype="f16", ragged=True, rotate=False),
        # long contexts, sixteen guesses each
        _tree("tree_32x8192_t16", B=32, lo=8192, hi=8192, T=16),
        # wide trees, wide groups, codes alone
        _tree("tree_5x20011_t33_noqjl", B=5, lo=14003, hi=20011, T=33, Hq=64, page=32, qjl=False),
        # the widest tree over a book
        _tree("tree_2x131072_t64", B=2, lo=131072, hi=131072, T=64, page=64),
        # one reader's long prompt, a sixteenth of it read
        _blocks("blocks_1x8192", top=32),
        # a batch of such
        _blocks("blocks_32x8192", B=32),
        # three queries a sequence, mixed lengths, heads of their own
        _blocks("blocks_13_ragged_t3_f16", B=13, lo=100, hi=30011, T=3, Hq=8, page=32, top=24, dtype="f16", rotate=False),
        # long contexts in large pages, wide groups
        _blocks("blocks_24x32768_p128", B=24, lo=32768, hi=32768, Hq=64, page=128, top=16),
        # books, small pages: the selection is most of the work
        _blocks("blocks_8x131072", B=8, lo=131072, hi=131072, top=256),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (16, 16), (8, 8), (64, 8), (16, 4), (7, 1), (40, 8), (10, 2)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    qjl, rotate = rng.random() < 0.8, rng.random() < 0.6
    if rng.random() < 0.5:
        T = _log(rng, 1, 64)
        B = _log(rng, 1, 64)
        # cached tokens times rows no more than the widest listed tree's
        most = min(131072, 262144 // B, 2 * 131072 * 64 * 32 // (B * T * Hq))
        hi = _log(rng, max(T, 20), max(T + 20, most))
        return _tree(None, dtype=dtype, Hq=Hq, Hkv=Hkv, B=B, lo=max(T, hi // rng.choice([1, 1, 3, 20])), hi=hi, page=page,
                     T=T, qjl=qjl, rotate=rotate, ragged=rng.random() < 0.4)
    B = _log(rng, 1, 64)
    hi = _log(rng, 100, min(131072, 1048576 // B))
    T = rng.choice([1, 1, 1, 2, 5])
    top = _log(rng, 2, max(2, min(256, 4096 // page)))
    return _blocks(None, dtype=dtype, Hq=Hq, Hkv=Hkv, B=B, lo=max(T, hi // rng.choice([1, 1, 3, 20])), hi=hi, page=page,
                   T=T, qjl=qjl, rotate=rotate, top=top)


# ── inputs ──────────────────────────────────────────────────────────────

def _lengths(case):
    """From lo to hi in equal steps, out of order."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + (hi - lo) * ((b * 7 + 3) % B) // max(1, B - 1) if B > 1 else hi for b in range(B)]


def _drafts(case):
    """Drafted tokens of each sequence."""
    T = case["T"]
    return [(b * 5 + T) % (T + 1) if case["ragged"] else T for b in range(case["B"])]


def _parents(case, seed):
    """int64 (B, T): a drafted token's parent among those before it, -1 where
    it follows the last cached token."""
    g = torch.Generator().manual_seed(seed + 1)
    B, T = case["B"], case["T"]
    back = torch.randint(1, 7, (B, T), generator=g) // 2 + 1         # 1 to 4 tokens before it
    return (torch.arange(T)[None, :] - back).clamp_min(-1)


def _hadamard(dtype):
    """The normalized Hadamard matrix: entry (i, j) has the sign of the parity of i & j's bits."""
    i = torch.arange(D, device=DEV)
    p = i[:, None] & i[None, :]
    odd = sum(((p >> k) & 1) for k in range(7)) % 2
    return (1.0 - 2.0 * odd.to(dtype)) / math.sqrt(D)


def _signs_matrix(Hkv):
    """float32 (Hkv, 64, 128): each head's +-1 projections, from the head's seed."""
    return torch.stack([torch.randint(0, 2, (D // 2, D), generator=torch.Generator().manual_seed((UID % 1024) ^ h),
                                      dtype=torch.float32) * 2 - 1 for h in range(Hkv)]).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    B, T, Hq, Hkv, page = case["B"], case["T"], case["Hq"], case["Hkv"], case["page"]
    lens = _lengths(case)
    need = [(n + page - 1) // page for n in lens]
    max_pages, n_pages = max(need) + 1, sum(need) + 3
    # the levels as a calibration finds them: a scale of its own for each head
    half = torch.tensor(_LEVELS)
    levels = torch.cat((-half.flip(0), half))
    cb = (levels[None, :] * (0.8 + 0.5 * torch.rand(Hkv, 1, generator=gc))).to(DEV)
    mid = ((levels[1:] + levels[:-1]) / 2).to(DEV)
    # codes of keys and values that the rotation has made Gaussian; the residuals' norms and signs as such keys leave them
    kn = torch.empty(n_pages, Hkv, page, D // 2, dtype=torch.uint8, device=DEV)
    vn = torch.empty_like(kn)
    for pool in (kn, vn):
        flat = pool.view(-1, D // 2)
        for at in range(0, flat.shape[0], 1 << 20):
            n = min(1 << 20, flat.shape[0] - at)
            code = torch.bucketize(torch.randn(n, D, generator=g, device=DEV), mid, out_int32=True).to(torch.uint8)
            flat[at:at + n] = code[:, 0::2] | (code[:, 1::2] << 4)
    kq = torch.randint(0, 256, (n_pages, Hkv, page, D // 16), generator=g, device=DEV, dtype=torch.uint8)
    kr = (1.1 + 0.07 * torch.randn(n_pages, Hkv, page, generator=g, device=DEV)) * (cb[:, 15] / 2.7326)[None, :, None]
    order = torch.randperm(n_pages, generator=gc)
    pt = torch.full((B, max_pages), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        pt[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    pt, seq_lens = pt.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    # queries: noise and, for every kv head, a part along one of its cached keys
    pos = (torch.rand(B, Hkv, generator=g, device=DEV) * seq_lens[:, None]).long().minimum(seq_lens[:, None].long() - 1)
    pg = pt.long().gather(1, pos // page)
    codes = _codes(kn[pg, torch.arange(Hkv, device=DEV)[None, :], pos % page])
    like = cb[torch.arange(Hkv, device=DEV)[None, :, None], codes]
    q = torch.randn(B, Hkv, Hq // Hkv, T, D, generator=g, device=DEV) + 0.35 * like[:, :, None, None, :]
    flip = None
    if case["rotate"]:
        flip = (torch.randint(0, 2, (D,), generator=gc) * 2 - 1).to(torch.int8).to(DEV)
        q = (q @ _hadamard(torch.float32)) * flip
    q = q.reshape(B, Hq, T, D).to(DTYPES[case["dtype"]]).contiguous()
    st = dict(case=case, q=q, kn=kn, kq=kq, kr=kr, vn=vn, cb=cb, flip=flip, pt=pt, lens=seq_lens, G=_signs_matrix(Hkv))
    if case["op"] == "tree":
        parents = _parents(case, seed)
        seen = torch.zeros(B, T, T + 1, dtype=torch.int64)           # [b, t, j]: t sees j; column T for "none"
        for t in range(T):
            up = seen.gather(1, parents[:, t].clamp_min(0)[:, None, None].expand(B, 1, T + 1))[:, 0] * (parents[:, t] >= 0)[:, None]
            up[:, t] = 1
            seen[:, t] = up
        weights = torch.tensor([1 << j if j < 63 else -(1 << 63) for j in range(T)], dtype=torch.int64)
        st.update(parents=parents, tree=(seen[:, :, :T] * weights).sum(-1).to(DEV),
                  n_draft=torch.tensor(_drafts(case), dtype=torch.int32, device=DEV))
    else:
        c = _codes(kn)
        # a page's last tokens may lie behind its sequence's end: bounds are of those before it
        used = torch.zeros(n_pages, dtype=torch.int64)
        for b, n in enumerate(need):
            used[pt[b, :n].cpu().long()] = torch.tensor([min(page, lens[b] - j * page) for j in range(n)])
        live = (torch.arange(page, device=DEV)[None, :] < used.to(DEV)[:, None])[:, None, :, None]
        lo = torch.empty(n_pages, Hkv, D, dtype=torch.uint8, device=DEV)
        hi = torch.empty_like(lo)
        step = max(1, (1 << 22) // (Hkv * page))
        del c
        for at in range(0, n_pages, step):
            c, m = _codes(kn[at:at + step]).to(torch.uint8), live[at:at + step]
            lo[at:at + step] = torch.where(m, c, 15).amin(2)
            hi[at:at + step] = torch.where(m, c, 0).amax(2)
        st.update(lo=lo, hi=hi)
    if own:
        from omnistack_rs.cache import PagedBlockAttention, PagedKVCache, PagedTreeAttention
        cache = PagedKVCache(n_pages, Hkv, page, device=DEV, bounds=case["op"] == "blocks")
        cache.k_nibbles, cache.k_qjl, cache.k_norms, cache.v_nibbles = kn, kq, kr, vn
        kw = dict(user_id=UID, with_qjl=case["qjl"], q_dtype=q.dtype, rotate_q=case["rotate"], sign_flip=flip, q_tokens=T)
        if case["op"] == "tree":
            st["handle"] = PagedTreeAttention(cache, cb, Hq, B, max_pages, **kw)
        else:
            cache.update_bounds(pt, torch.zeros_like(seq_lens), seq_lens)
            st["handle"] = PagedBlockAttention(cache, cb, Hq, B, max_pages, case["top"], **kw)
    return st


# ── the plain forms ─────────────────────────────────────────────────────

def _codes(packed):
    """int64 codes of packed nibbles, (..., 64) uint8 to (..., 128)."""
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2).long()


def _keys(st, pages):
    """float32 keys of whole pages, from page ids (..., P) per head: (..., Hkv, P, page, 128)
    where `pages` is (..., Hkv, P)."""
    heads = torch.arange(st["cb"].shape[0], device=DEV)[:, None]
    k = st["cb"][heads[..., None, None], _codes(st["kn"][pages, heads])]
    if st["case"]["qjl"]:
        byte = st["kq"][pages, heads]
        sign = ((byte[..., None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1).flatten(-2).float() * 2 - 1
        k = k + (sign @ st["G"][:, None]) * (st["kr"][pages, heads] * (math.sqrt(2 / math.pi) / D))[..., None]
    return k


def _values(st, pages):
    heads = torch.arange(st["cb"].shape[0], device=DEV)[:, None]
    return st["cb"][heads[..., None, None], _codes(st["vn"][pages, heads])]


def _softmax(s, visible):
    s = torch.where(visible, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _rotated(st, q):
    return (q * st["flip"]) @ _hadamard(q.dtype) if st["flip"] is not None else q


def _run_tree(st):
    case, B, T = st["case"], st["case"]["B"], st["case"]["T"]
    Hkv, G = case["Hkv"], case["Hq"] // case["Hkv"]
    pages = st["pt"].long().clamp_min(0)[:, None, :].expand(B, Hkv, -1)
    k, v = _keys(st, pages).flatten(2, 3), _values(st, pages).flatten(2, 3)
    pos = torch.arange(k.shape[2], device=DEV)
    base = (st["lens"] - st["n_draft"])[:, None, None]
    bit = (st["tree"][:, :, None] >> (pos - base).clamp(0, 63)) & 1
    visible = (pos < base) | ((bit == 1) & (pos < st["lens"][:, None, None]))             # (B, T, S)
    q = _rotated(st, st["q"].float()).view(B, Hkv, G, T, D)
    s = (q.reshape(B, Hkv, G * T, D) @ k.transpose(-1, -2)).view(B, Hkv, G, T, -1) * SCALE
    p = _softmax(s, visible[:, None, None])
    o = (p.view(B, Hkv, G * T, -1) @ v).view(B, Hkv * G, T, D)
    drafted = torch.arange(T, device=DEV)[None, :] < st["n_draft"][:, None]
    return torch.where(drafted[:, None, :, None], o, 0.0).to(st["q"].dtype)


def _whole(x, dim):
    """float64 x times the power of two that brings the largest of `dim` into [64, 128), rounded to whole numbers."""
    bits = x.abs().amax(dim, keepdim=True).view(torch.int64) >> 52                                # exponents, biased by 1023
    return torch.round(x * ((2 * 1023 + 6 - bits) << 52).view(torch.float64)).clamp(-127, 127)


def _run_blocks(st):
    case, B, T, page, top = st["case"], st["case"]["B"], st["case"]["T"], st["case"]["page"], st["case"]["top"]
    Hkv, G = case["Hkv"], case["Hq"] // case["Hkv"]
    # the score in whole numbers, from exact sums: float64 of 16-bit values, the transform's factor left off
    q64 = st["q"].double()
    if st["flip"] is not None:
        q64 = (q64 * st["flip"]) @ torch.sign(_hadamard(torch.float64))
    q64 = q64.view(B, Hkv, G, T, D)
    Q = _whole(torch.cat((q64.clamp_min(0).sum(2), (-q64).clamp_min(0).sum(2)), -1), -1)          # (B, Hkv, T, 256)
    c = _whole(st["cb"].double(), -1).float()                                                     # (Hkv, 16)
    pages = st["pt"].long().clamp_min(0)
    heads = torch.arange(Hkv, device=DEV)
    edge = torch.cat((c[heads[:, None], st["hi"].long()], -c[heads[:, None], st["lo"].long()]), -1)   # (n_pages, Hkv, 256)
    score = Q.float() @ edge[pages].permute(0, 2, 3, 1)                                           # (B, Hkv, T, P), below 2^23
    seen = st["lens"][:, None].long() - T + 1 + torch.arange(T, device=DEV)                       # (B, T) visible tokens
    n = ((seen + page - 1) // page)[:, None, :, None]
    j = torch.arange(pages.shape[1], device=DEV)
    score = torch.where((j == 0) | (j == n - 1), math.inf, score)
    score = torch.where(j < n, score, -math.inf)
    score = torch.nn.functional.pad(score, (0, max(0, top - score.shape[-1])), value=-math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :top]                      # ties: the lowest index
    best = torch.where(best < n, best, 1 << 30).sort(-1)[0]
    blocks = torch.where(best < 1 << 30, best, -1)
    ids = pages[:, None, None, :].expand(B, Hkv, T, -1).gather(-1, blocks.clamp_min(0))           # (B, Hkv, T, top)
    ids = ids.transpose(1, 2)                                                                     # (B, T, Hkv, top)
    k, v = _keys(st, ids).flatten(3, 4), _values(st, ids).flatten(3, 4)
    pos = (blocks.transpose(1, 2)[..., None] * page + torch.arange(page, device=DEV)).flatten(3, 4)
    visible = (pos >= 0) & (pos < seen[:, :, None, None])
    q = _rotated(st, st["q"].float()).view(B, Hkv, G, T, D).permute(0, 3, 1, 2, 4)
    p = _softmax((q @ k.transpose(-1, -2)) * SCALE, visible[..., None, :])
    o = (p @ v).permute(0, 2, 3, 1, 4).reshape(B, Hkv * G, T, D)
    return {"out": o.to(st["q"].dtype), "blocks": blocks.int()}


def run(st):
    tree = st["case"]["op"] == "tree"
    if own:
        if tree:
            return st["handle"].run(st["q"], st["pt"], st["lens"], st["tree"], st["n_draft"])
        out = st["handle"].run(st["q"], st["pt"], st["lens"])
        return {"out": out, "blocks": st["handle"].blocks}
    return _run_tree(st) if tree else _run_blocks(st)


# ── what a pass cannot do without ───────────────────────────────────────

def work(case):
    B, T, Hq, Hkv, page = case["B"], case["T"], case["Hq"], case["Hkv"], case["page"]
    per_token, per_pair = (140, 5 * D) if case["qjl"] else (128, 4 * D)
    lens = _lengths(case)
    nbytes = 2 * 2 * B * Hq * T * D + 4 * sum((n + page - 1) // page for n in lens)
    flops = 0
    if case["op"] == "tree":
        for n, d in zip(lens, _drafts(case)):
            if d:
                nbytes += n * Hkv * per_token
                flops += per_pair * Hq * d * (n - d)         # the tree's own pairs are few
        return dict(bytes=nbytes + 8 * B * T, flops=flops)
    for n in lens:
        for t in range(T):
            seen = n - T + 1 + t
            some = min(seen, case["top"] * page)
            flops += per_pair * Hq * some + 4 * D * Hkv * ((seen + page - 1) // page)
            nbytes += 4 * Hkv * case["top"]
        # queries of one sequence may select the same blocks: these are counted once
        nbytes += Hkv * (D * ((n + page - 1) // page) + per_token * min(n, case["top"] * page))
    return dict(bytes=nbytes, flops=flops)


# ── the definition in 64 bits ───────────────────────────────────────────

def exact(case, seed):
    """Sequence by sequence, head by head: each visible token's key and value
    spelled out in float64, from the tree's parents and whole-number scores."""
    st = prepare(case, seed)
    B, T, Hkv, page = case["B"], case["T"], case["Hkv"], case["page"]
    G = case["Hq"] // Hkv
    lens, pt = _lengths(case), st["pt"].long()
    cb = st["cb"].double()
    factor = math.sqrt(2.0 / math.pi) / D
    q = st["q"].double()
    unscaled = q
    if st["flip"] is not None:
        odd = torch.tensor([[bin(i & j).count("1") % 2 for j in range(D)] for i in range(D)], device=DEV)
        unscaled = (q * st["flip"].double()) @ (1.0 - 2.0 * odd.double())
        q = unscaled / math.sqrt(128.0)
    out = torch.zeros(B, case["Hq"], T, D, dtype=torch.float64, device=DEV)

    def attend(b, h, rows, tokens, hidden=None):
        """Rows (n, 128) of head h over tokens at positions `tokens`."""
        total, peak = 0.0, torch.full((rows.shape[0], 1), -math.inf, dtype=torch.float64, device=DEV)
        acc = torch.zeros(rows.shape[0], D, dtype=torch.float64, device=DEV)
        for at in range(0, tokens.numel(), 1 << 16):
            tok = tokens[at:at + (1 << 16)]
            where = (pt[b, tok // page], h, tok % page)
            raw = st["kn"][where].to(torch.int64)
            key = torch.empty(tok.numel(), D, dtype=torch.float64, device=DEV)
            key[:, 0::2], key[:, 1::2] = cb[h][raw % 16], cb[h][raw // 16]
            if case["qjl"]:
                byte = st["kq"][where].to(torch.int64)
                bits = torch.stack([(byte // (1 << i)) % 2 for i in range(8)], 2).reshape(tok.numel(), D // 2)
                key += (2.0 * bits.double() - 1.0) @ st["G"][h].double() * (st["kr"][where].double() * factor)[:, None]
            raw = st["vn"][where].to(torch.int64)
            value = torch.empty_like(key)
            value[:, 0::2], value[:, 1::2] = cb[h][raw % 16], cb[h][raw // 16]
            s = rows @ key.T / math.sqrt(128.0)
            if hidden is not None:
                s = s.masked_fill(hidden[:, at:at + (1 << 16)], -math.inf)
            new = torch.maximum(peak, s.amax(1, keepdim=True))
            keep, w = torch.exp(peak - new), torch.exp(s - new)
            total, acc, peak = total * keep + w.sum(1, keepdim=True), acc * keep + w @ value, new
        return acc / total

    if case["op"] == "tree":
        drafts, parents = _drafts(case), st["parents"].tolist()
        for b in range(B):
            n, first = drafts[b], lens[b] - drafts[b]
            if not n:
                continue
            hidden = torch.zeros(n, lens[b], dtype=torch.bool)
            hidden[:, first:] = True
            for t in range(n):
                up = t
                while up >= 0:
                    hidden[t, first + up] = False
                    up = parents[b][up]
            hidden = hidden.to(DEV).repeat(G, 1)
            tokens = torch.arange(lens[b], device=DEV)
            for h in range(Hkv):
                rows = q[b, h * G:(h + 1) * G, :n].reshape(G * n, D)
                out[b, h * G:(h + 1) * G, :n] = attend(b, h, rows, tokens, hidden).view(G, n, D)
        return out

    top = case["top"]

    def whole(x):
        most = float(x.abs().max())
        return torch.round(x * 2.0 ** (7 - math.frexp(most)[1])).clamp(-127, 127).long()

    for b in range(B):
        for t in range(T):
            seen = lens[b] - T + 1 + t
            n = (seen + page - 1) // page
            for h in range(Hkv):
                heads = unscaled[b, h * G:(h + 1) * G, t]
                Q = whole(torch.stack((heads.clamp_min(0).sum(0), heads.clamp_max(0).sum(0))))
                c = whole(cb[h])
                ids = pt[b, :n]
                score = (c[st["hi"][ids, h].long()] * Q[0]).sum(1) + (c[st["lo"][ids, h].long()] * Q[1]).sum(1)
                # the index breaks ties: one whole number orders them all
                order = score * (1 << 24) - torch.arange(n, device=DEV)
                order[0] = order[n - 1] = 1 << 62
                chosen = torch.topk(order, min(top, n))[1].sort()[0]
                tokens = (chosen[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
                out[b, h * G:(h + 1) * G, t] = attend(b, h, q[b, h * G:(h + 1) * G, t], tokens[tokens < seen])
    return {"out": out, "blocks": None}
