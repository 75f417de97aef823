"""Attention of drafted tokens' trees over the paged cache (omni_attn_tree) and
the move of accepted ones (omni_cache_keep), against 64-bit forms."""
import math

import pytest
import torch

from tests import _pages as P

pytestmark = pytest.mark.gpu


def _q(B, Hq, T, seed, dtype, size=1.0):
    return (size * torch.randn(B, Hq, T, 128, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _want(q, parts, cb, uid, lens, drafts, tree, scale, with_qjl, rotate=False, flip=None):
    """float64 (result, bound) of paged_tree_attention."""
    B, Hq, T, _ = q.shape
    k, v = P.keys_values(*parts, cb, uid, with_qjl)
    H = k.shape[1]
    G = Hq // H
    x = P.rotated(q, flip) if rotate else q.double()
    want, bound = torch.zeros(B, Hq, T, 128).double(), torch.zeros(B, Hq, T, 128).double()
    for b in range(B):
        L, n = lens[b], drafts[b]
        if n == 0:
            continue
        row = tree[b] if tree.dim() == 2 else tree
        vis = torch.zeros(n, L, dtype=torch.bool)
        vis[:, :L - n] = True
        for t in range(n):
            for j in range(n):
                vis[t, L - n + j] = bool((int(row[t]) >> j) & 1)
        for h in range(Hq):
            o, e = P.attend(x[b, h, :n], k[b, h // G, :L], v[b, h // G, :L], vis, scale, q.dtype, rotate)
            want[b, h, :n], bound[b, h, :n] = o, e
    return want, bound


CASES = [
    # B, Hq, H, T, lens, drafts, page, dtype, qjl, rotate
    (1, 4, 4, 1, [1], None, 16, torch.bfloat16, True, False),
    (3, 8, 2, 5, [5, 6, 133], None, 16, torch.bfloat16, True, False),
    (4, 8, 2, 4, [4, 37, 16, 300], [0, 1, 4, 3], 32, torch.bfloat16, True, True),
    (2, 16, 16, 12, [31, 290], None, 64, torch.float16, True, True),
    (2, 10, 2, 9, [64, 65], [9, 2], 16, torch.float16, False, False),
    (1, 7, 1, 33, [1000], None, 128, torch.bfloat16, False, True),
    (2, 16, 2, 64, [64, 2100], [64, 63], 256, torch.bfloat16, True, False),
    (2, 32, 8, 16, [515, 3001], None, 1024, torch.float16, True, False),
    (1, 64, 1, 3, [97], None, 16, torch.bfloat16, True, False),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_tree_attention_against_64_bits(device, case, scale):
    from omnistack_rs.cache import PagedTreeAttention, paged_tree_attention, tree_masks
    B, Hq, H, T, lens, drafts, page, dtype, qjl, rotate = case
    uid = 5
    parts = P.packed(B, H, max(lens), seed=71)
    cb = P.codebooks(H)
    q = _q(B, Hq, T, 72, dtype, 1.5)
    flip = (torch.randint(0, 2, (128,), generator=torch.Generator().manual_seed(3)) * 2 - 1).to(torch.int8)
    tree = tree_masks(P.random_parents(B, T, 74))
    cache, pt, lt = P.paged(device, parts, page, lens, seed=page)
    nd = None if drafts is None else torch.tensor(drafts, dtype=torch.int32, device=device)
    kw = dict(user_id=uid, scale=scale, with_qjl=qjl, rotate_q=rotate, sign_flip=flip.to(device))
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), n_draft=nd, **kw)
    want, bound = _want(q, parts, cb, uid, lens, drafts or [T] * B, tree, 1 / math.sqrt(128) if scale is None else scale, qjl,
                        rotate, flip)
    assert got.dtype == dtype
    P.close(got, want, bound, str(case))
    # the prepared form, a wider table: the same numbers from another plan of splits
    wide = torch.full((B, pt.shape[1] + 40), -1, dtype=torch.int32, device=device)
    wide[:, :pt.shape[1]] = pt
    att = PagedTreeAttention(cache, cb.to(device), Hq, B, wide.shape[1], T, q_dtype=dtype, **kw)
    P.close(att.run(q.to(device), wide, lt, tree.to(device), nd), want, bound, f"prepared {case}")


def test_one_tree_for_all_and_one_codebook(device):
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, Hq, H, T, lens = 3, 8, 4, 6, [6, 50, 77]
    parts, cb, q = P.packed(B, H, 77, seed=81), P.codebooks(1)[0], _q(B, Hq, T, 82, torch.bfloat16)
    tree = tree_masks(torch.tensor([-1, 0, 0, 1, -1, 4]))
    cache, pt, lt = P.paged(device, parts, 16, lens)
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), user_id=9)
    want, bound = _want(q, parts, cb, 9, lens, [T] * B, tree, 1 / math.sqrt(128), True)
    P.close(got, want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_tokens_reach_nobody(device, dtype):
    """NaN, infinities and other codes in tokens that a row does not see leave
    its bits alone: drafted tokens off its path, slots behind the sequence, page
    entries behind its last page."""
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, Hq, H, T, L = 1, 8, 2, 20, 61
    parts = P.packed(B, H, L, seed=91)
    q, cb = _q(B, Hq, T, 92, dtype), P.codebooks(H)
    parents = P.random_parents(B, T, 93)
    tree = tree_masks(parents)
    cache, pt, lt = P.paged(device, parts, 16, [L])
    args = (q.to(device), cache, pt, lt, cb.to(device), tree.to(device))
    ref = paged_tree_attention(*args)
    assert torch.isfinite(ref).all()
    cache.k_norms[pt[0, -1].long(), :, L % 16:] = float("nan")
    cache.v_nibbles[pt[0, -1].long(), :, L % 16:] = 0xF0
    assert torch.equal(paged_tree_attention(*args), ref)
    for j, bad in ((0, float("nan")), (7, float("inf")), (13, float("-inf")), (19, 3.0e38)):
        pos = L - T + j
        keep = cache.k_norms[pt[0, pos // 16].long(), :, pos % 16].clone()
        nib = cache.k_nibbles[pt[0, pos // 16].long(), :, pos % 16].clone()
        cache.k_norms[pt[0, pos // 16].long(), :, pos % 16] = bad
        cache.k_nibbles[pt[0, pos // 16].long(), :, pos % 16] ^= 0x5A
        got = paged_tree_attention(*args)
        sees = torch.tensor([(int(tree[0, t]) >> j) & 1 for t in range(T)], dtype=torch.bool)
        assert torch.equal(got[:, :, ~sees], ref[:, :, ~sees]), f"hidden token {j}"
        assert not torch.equal(got[:, :, sees], ref[:, :, sees]), f"visible token {j}"
        cache.k_norms[pt[0, pos // 16].long(), :, pos % 16] = keep
        cache.k_nibbles[pt[0, pos // 16].long(), :, pos % 16] = nib
    assert torch.equal(paged_tree_attention(*args), ref)


def test_rows_that_see_nothing_bad_lengths_and_bad_pages(device):
    from omnistack_rs.cache import paged_tree_attention
    B, Hq, H, T = 6, 8, 2, 3
    lens = [3, 40, 0, 50, 33, 48]
    parts = P.packed(B, H, 50, seed=95)
    q, cb = _q(B, Hq, T, 96, torch.bfloat16), P.codebooks(H)
    cache, pt, lt = P.paged(device, parts, 16, lens)
    tree = torch.tensor([[0, 2, 7]] * B)                     # the first row sees no drafted token, itself included
    nd = torch.tensor([3, 3, 0, 4, 3, 3], dtype=torch.int32)
    pt[4, 1] = cache.n_pages
    lt[5] = pt.shape[1] * 16 + 1
    args = (q.to(device), cache, pt, lt, cb.to(device), tree.to(device))
    for n, error in ((nd, ValueError), (nd.clamp_max(3), ValueError)):
        with pytest.raises(error):
            paged_tree_attention(*args, n_draft=n.to(device))
    got = paged_tree_attention(*args, n_draft=nd.to(device), validate=False).cpu()
    assert torch.isnan(got[0, :, 0]).all() and torch.isfinite(got[0, :, 1:]).all()      # nothing cached before the tree
    assert torch.isfinite(got[1]).all()
    assert (got[2] == 0).all()                                                          # nothing drafted
    assert torch.isnan(got[3:]).all()             # more drafted than T; a page outside the pool; a length past the table
    lt[5], pt[4, 1] = 48, -1
    with pytest.raises(IndexError):
        paged_tree_attention(*args, n_draft=nd.clamp_max(3).to(device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_of_a_query(device, dtype):
    """Rows with NaN or an infinity are NaN (an infinite score minus itself), large and small rows are exact to their own
    scale, and no row touches another."""
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, Hq, H, T, L = 1, 16, 2, 4, 200
    parts, cb = P.packed(B, H, L, seed=101), P.codebooks(H)
    q = _q(B, Hq, T, 102, dtype)
    q[0, 3, 1, 5] = float("nan")
    q[0, 9, 2, 0] = float("inf")
    q[0, 1] *= 1e-4
    q[0, 12] *= 60.0
    q[0, 15, 3] = 0.0
    tree = tree_masks(torch.tensor([-1, 0, 1, 2]))
    cache, pt, lt = P.paged(device, parts, 16, [L])
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device)).cpu()
    ok = torch.ones(Hq, T, dtype=torch.bool)
    ok[3, 1] = ok[9, 2] = False
    assert torch.isnan(got[0][~ok]).all()
    clean = torch.where(torch.isfinite(q), q, 0.0)
    want, bound = _want(clean, parts, cb, 0, [L], [T], tree, 1 / math.sqrt(128), True)
    P.close(got[0][ok], want[0][ok], bound[0][ok])


def test_scale_zero_and_codebook_sizes(device):
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, Hq, H, T, L = 1, 8, 2, 2, 77
    parts, q = P.packed(B, H, L, seed=105), _q(B, Hq, T, 106, torch.float16)
    tree = tree_masks(torch.tensor([-1, 0]))
    cache, pt, lt = P.paged(device, parts, 16, [L])
    for size, scale in ((1.0, 0.0), (1e-12, 1.0), (2e5, 1e-6), (1e20, 1e-21)):
        cb = P.codebooks(H) * size
        cache.k_norms.zero_()
        zero = (*parts[:2], torch.zeros_like(parts[2]), parts[3])
        got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), scale=scale).cpu()
        want, bound = _want(q, zero, cb, 0, [L], [T], tree, scale, True)
        # fp16 holds from 2^-24 to 65504
        want, bound = want.clamp(-1e30, 1e30), bound + 2.0 ** -24
        big = want.abs() > 65000
        P.close(torch.where(big, 0.0, got.double()), torch.where(big, 0.0, want), bound, f"{size} {scale}")


def test_chain_equals_causal_attention_and_splits(device):
    """A chain of drafted tokens is paged_attention's causal form (fp32, another
    kernel), for a long sequence that is split and merged."""
    from omnistack_rs.cache import paged_attention, paged_tree_attention, tree_masks
    B, Hq, H, T, L, uid = 1, 32, 8, 8, 20011, 3
    parts, cb = P.packed(B, H, L, seed=111), P.codebooks(H)
    q = _q(B, Hq, T, 112, torch.bfloat16, 3.0).to(device)
    cache, pt, lt = P.paged(device, parts, 64, [L])
    tree = tree_masks(torch.arange(-1, T - 1)).to(device)
    got = paged_tree_attention(q, cache, pt, lt, cb.to(device), tree, user_id=uid)
    want, bound = _want(q.cpu(), parts, cb, uid, [L], [T], tree.cpu(), 1 / math.sqrt(128), True)
    P.close(got, want, bound)
    ref = paged_attention(q, cache, pt, lt, cb.to(device), user_id=uid, causal=True)
    P.close(got, ref.double().cpu(), bound + 2e-3, "causal")        # paged_attention's own bar
    again = paged_tree_attention(q, cache, pt, lt, cb.to(device), tree, user_id=uid)
    assert torch.equal(got, again)


def test_strides_streams_and_capture(device):
    """q as a transposed view, off 16 bytes, on another stream; the prepared
    form captured, replayed on new inputs and against eager calls between."""
    from omnistack_rs.cache import PagedTreeAttention, paged_tree_attention, tree_masks
    B, Hq, H, T, lens = 4, 16, 4, 6, [100, 10, 333, 64]
    parts, cb = P.packed(B, H, 333, seed=121), P.codebooks(H).to(device)
    q = _q(B, Hq, T, 122, torch.bfloat16).to(device)
    tree = tree_masks(P.random_parents(B, T, 123)).to(device)
    cache, pt, lt = P.paged(device, parts, 32, lens)
    ref = paged_tree_attention(q, cache, pt, lt, cb, tree)
    view = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert not view.is_contiguous() and torch.equal(paged_tree_attention(view, cache, pt, lt, cb, tree), ref)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape).copy_(q)
    assert torch.equal(paged_tree_attention(odd, cache, pt, lt, cb, tree), ref)
    att = PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], T)
    with pytest.raises(ValueError):
        att.run(odd, pt, lt, tree)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(att.run(q, pt, lt, tree), ref)
    torch.cuda.synchronize()
    qs, ls = q.clone(), lt.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = att.run(qs, pt, ls, tree)
    for k in range(4):
        qs.copy_(_q(B, Hq, T, 130 + k, torch.bfloat16))
        ls.copy_(lt - k)
        want = paged_tree_attention(qs, cache, pt, ls, cb, tree)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {k}"
        torch.zeros(1 << 20, device=device).sum().item()


def test_drafting_loop(device):
    """Append drafted tokens, attend to their tree, keep an accepted path: the
    cache is then that of the accepted tokens appended alone, bounds included."""
    from omnistack_rs.cache import PagedKVCache, paged_tree_attention, tree_masks
    from omnistack_rs.kernels.quantize import PackedKVEncoder
    B, Hq, H, T, uid = 3, 8, 2, 10, 4
    cb = P.codebooks(H).to(device)
    enc = PackedKVEncoder(cb, H, user_id=uid, dtype=torch.bfloat16, device=device)
    caches = [PagedKVCache(40, H, 16, device=device, bounds=True) for _ in range(2)]
    g = torch.Generator().manual_seed(7)
    lens = torch.tensor([13, 32, 47], dtype=torch.int32)
    tables = []
    for c in caches:
        tables.append(c.page_table([c.allocate(64 + 32) for _ in range(B)]))
    zero = torch.zeros(B, dtype=torch.int32, device=device)
    k, v = (torch.randn(B, H, 47, 128, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    for c, pt in zip(caches, tables):
        c.append(enc, k, v, pt, zero)                          # the longest prompt's tokens; shorter ones are overwritten
    for step, accepted in enumerate(([[0, 2, 5, 9], [1], []], [[3, 4], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9], [2, 7]])):
        dk, dv = (torch.randn(B, H, T, 128, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
        at = lens.to(device)
        caches[0].append(enc, dk, dv, tables[0], at)
        tree = tree_masks(P.random_parents(B, T, 5 + step)).to(device)
        q = _q(B, Hq, T, 8 + step, torch.bfloat16).to(device)
        o = paged_tree_attention(q, caches[0], tables[0], at + T, cb, tree, user_id=uid)
        assert torch.isfinite(o).all()
        kept = torch.full((B, T), -1, dtype=torch.int32)
        for b, path in enumerate(accepted):
            kept[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
        caches[0].keep(tables[0], at, kept.to(device))
        for b, path in enumerate(accepted):
            if path:
                one = slice(b, b + 1)
                caches[1].append(enc, dk[one][:, :, path].contiguous(), dv[one][:, :, path].contiguous(),
                                 tables[1][one].contiguous(), at[one].contiguous())
        lens = lens + torch.tensor([len(p) for p in accepted], dtype=torch.int32)
        for b in range(B):
            for p in range(0, int(lens[b]), 16):
                n, i, j = min(16, int(lens[b]) - p), int(tables[0][b, p // 16]), int(tables[1][b, p // 16])
                for name in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles"):
                    assert torch.equal(getattr(caches[0], name)[i, :, :n], getattr(caches[1], name)[j, :, :n]), (name, step, b, p)
                c = P.codes(caches[0].k_nibbles[i, :, :n].cpu())
                want = c.amin(1) | (c.amax(1) << 4)
                if int(lens[b]) - p <= 16:                      # the last page
                    assert torch.equal(caches[0].k_bounds[i].cpu().long(), want), (step, b, p)


def test_keep_any_order_and_outside(device):
    from omnistack_rs.cache import PagedKVCache
    H = 3
    cache = PagedKVCache(6, H, 16, device=device)
    for name in ("k_nibbles", "k_qjl", "v_nibbles"):
        getattr(cache, name).random_(0, 256)
    cache.k_norms.uniform_()
    before = {n: getattr(cache, n).clone() for n in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles")}
    pt = torch.tensor([[2, 0, 4], [1, 7, 3]], dtype=torch.int32, device=device)
    pos = torch.tensor([10, 12], dtype=torch.int32, device=device)
    kept = torch.tensor([[5, 0, 3, 63, 9], [2, -1, 1, 0, 70]], dtype=torch.int32, device=device)
    with pytest.raises(ValueError):
        cache.keep(pt, pos, kept)                               # 63 lies past the table, 70 past any tree
    with pytest.raises(IndexError):
        cache.keep(pt, pos, kept.clamp(-1, 9))                  # page 7
    cache.keep(pt, pos, kept, validate=False)
    tok = lambda b, p: (int(pt[b, p // 16]), slice(None), p % 16)  # noqa: E731
    want = {n: t.clone() for n, t in before.items()}
    for b, moves in ((0, [(5, 0), (0, 1), (3, 2), (9, 4)]), (1, [(2, 0), (1, 2), (0, 3)])):
        for frm, to in moves:
            for n in want:
                want[n][tok(b, int(pos[b]) + to)] = before[n][tok(b, int(pos[b]) + frm)]
    for n in want:
        assert torch.equal(getattr(cache, n), want[n]), n


def test_refusals(device):
    from omnistack_rs.cache import PagedTreeAttention, paged_tree_attention
    B, Hq, H, T = 2, 8, 2, 4
    parts, cb = P.packed(B, H, 40, seed=141), P.codebooks(H).to(device)
    cache, pt, lt = P.paged(device, parts, 16)
    q = _q(B, Hq, T, 142, torch.bfloat16).to(device)
    tree = torch.full((B, T), 1, dtype=torch.int64, device=device)
    ok = lambda **kw: paged_tree_attention(*[kw.get(n, d) for n, d in  # noqa: E731
                                             (("q", q), ("cache", cache), ("pt", pt), ("lens", lt), ("cb", cb), ("tree", tree))],
                                           **kw.get("more", {}))
    ok()
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(tree=tree.int()),
                dict(tree=tree[:, :3]), dict(pt=pt[:1]), dict(lens=lt[:1]), dict(cb=cb[:, :8]),
                dict(more=dict(scale=float("inf"))), dict(more=dict(n_draft=torch.tensor([1], device=device))),
                dict(more=dict(n_draft=torch.tensor([1, 5], device=device))),
                dict(q=q.repeat(1, 1, 17, 1), tree=tree.repeat(1, 17))):
        with pytest.raises(ValueError):
            ok(**bad)
    with pytest.raises(RuntimeError):
        ok(tree=tree.cpu())
    with pytest.raises(ValueError):
        PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], 65)
    with pytest.raises(ValueError):
        PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], T, q_dtype=torch.float32)
    att = PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], T)
    for args in ((q[:1], pt, lt, tree), (q, pt.long(), lt, tree), (q, pt, lt.long(), tree), (q, pt, lt, tree.int()),
                 (q.half(), pt, lt, tree), (q, pt, lt, tree, torch.tensor([1, 2], device=device))):
        with pytest.raises(ValueError):
            att.run(*args)
    empty = paged_tree_attention(q[:0], cache, pt[:0], lt[:0], cb, tree[:0])
    assert empty.shape == (0, Hq, T, 128)
