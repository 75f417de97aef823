"""The attention over drafted tokens' trees and selected blocks in calls that
fill the chip: every number of query rows a block, lists short and long, merged
splits; the selection's other paths; large pools; calls that overlap."""
import math

import pytest
import torch

from tests import _pages as P

pytestmark = pytest.mark.gpu


def _q(B, Hq, T, seed, dtype):
    return torch.randn(B, Hq, T, 128, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _visible(tree, n, L):
    vis = torch.zeros(n, L, dtype=torch.bool)
    vis[:, :L - n] = True
    for t in range(n):
        for j in range(n):
            vis[t, L - n + j] = bool((int(tree[t]) >> j) & 1)
    return vis


def _tree_want(q, parts, cb, uid, lens, tree, qjl):
    """float64 (result, bound): a kv head's query heads together."""
    B, Hq, T, _ = q.shape
    k, v = P.keys_values(*parts, cb, uid, qjl)
    H = k.shape[1]
    G = Hq // H
    want, bound = torch.zeros(B, Hq, T, 128).double(), torch.zeros(B, Hq, T, 128).double()
    for b in range(B):
        vis = _visible(tree[b], T, lens[b]).repeat(G, 1)
        for h in range(H):
            o, e = P.attend(q[b, h * G:(h + 1) * G].double().reshape(G * T, 128), k[b, h, :lens[b]], v[b, h, :lens[b]], vis,
                            1 / math.sqrt(128), q.dtype, False)
            want[b, h * G:(h + 1) * G], bound[b, h * G:(h + 1) * G] = o.view(G, T, 128), e.view(G, T, 128)
    return want, bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("qjl", [True, False])
@pytest.mark.parametrize("G,T", [(4, 4), (4, 5), (4, 8), (4, 12), (4, 16), (5, 33)])
def test_rows_of_a_block(device, G, T, qjl, dtype):
    """1 to 165 query rows a list, 256 lists."""
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, H, uid = 32, 8, 4
    lens = [T + (b * 37) % 150 for b in range(B)]
    parts, cb = P.packed(B, H, max(lens), seed=301), P.codebooks(H)
    q, tree = _q(B, G * H, T, 302, dtype), tree_masks(P.random_parents(B, T, 303))
    cache, pt, lt = P.paged(device, parts, 16, lens)
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), user_id=uid, with_qjl=qjl)
    want, bound = _tree_want(q, parts, cb, uid, lens, tree, qjl)
    P.close(got, want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("qjl", [True, False])
@pytest.mark.parametrize("G,T,most", [(4, 8, 192), (3, 7, 60), (17, 1, 33), (1, 3, 500)])
def test_more_short_lists_than_compute_units(device, G, T, most, qjl, dtype):
    """600 lists of up to six tiles, 3 to 32 rows each, some of their sequences without drafted tokens or with fewer."""
    from omnistack_rs.cache import paged_tree_attention, tree_masks
    B, H, uid = 75, 8, 4
    lens = [T + (b * 37) % (most - T + 1) for b in range(B)]
    parts, cb = P.packed(B, H, max(lens), seed=371), P.codebooks(H)
    q, tree = _q(B, G * H, T, 372, dtype), tree_masks(P.random_parents(B, T, 373))
    cache, pt, lt = P.paged(device, parts, 16, lens)
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), user_id=uid, with_qjl=qjl)
    want, bound = _tree_want(q, parts, cb, uid, lens, tree, qjl)
    P.close(got, want, bound)
    drafts = torch.tensor([(b * 3) % (T + 1) for b in range(B)], dtype=torch.int32, device=device)
    some = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), user_id=uid, with_qjl=qjl,
                                n_draft=drafts)
    for b, n in enumerate(drafts.tolist()):
        assert (some[b, :, n:] == 0).all() and torch.isfinite(some[b, :, :n]).all()
        if n == T:
            assert torch.equal(some[b], got[b])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,G,T,L", [(32, 8, 1, 4, 2200), (2, 8, 4, 16, 4111), (2, 4, 4, 8, 5000), (1, 3, 8, 6, 7001)])
def test_long_lists(device, B, H, G, T, L, dtype):
    """More than 64 tiles a block, whole or in merged splits; centroids off center, which long sums of V would show."""
    from omnistack_rs.cache import PagedTreeAttention, tree_masks
    lens = [L - (b * 613) % (L // 2) for b in range(B)]
    parts, cb = P.packed(B, H, L, seed=311), P.codebooks(H) + 1.7
    q, tree = _q(B, G * H, T, 312, dtype), tree_masks(P.random_parents(B, T, 313))
    cache, pt, lt = P.paged(device, parts, 32, lens)
    att = PagedTreeAttention(cache, cb.to(device), G * H, B, pt.shape[1], T, user_id=9, q_dtype=dtype)
    got = att.run(q.to(device), pt, lt, tree.to(device))
    want, bound = _tree_want(q, parts, cb, 9, lens, tree, True)
    P.close(got, want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,G,T,page,top", [(16, 4, 20, 4, 16, 5), (16, 4, 40, 4, 32, 3), (16, 4, 64, 4, 16, 4), (16, 8, 2, 2, 64, 40),
                                              (1, 2, 4, 1, 128, 30), (20, 4, 24, 4, 32, 5), (35, 8, 3, 1, 16, 7)])
def test_selected_blocks_rows(device, B, H, G, T, page, top, dtype):
    """Many heads a group, long selections, a selection in merged splits."""
    from omnistack_rs.cache import paged_block_attention
    n = top + 6
    L, uid = n * page - 5, 8
    parts, cb = P.packed(B, H, L, seed=321), P.codebooks(H)
    q = _q(B, G * H, T, 322, dtype)
    cache, pt, lt = P.paged(device, parts, page)
    g = torch.Generator().manual_seed(323)
    blocks = torch.stack([torch.randperm(n, generator=g)[:top] for _ in range(B * H * T)]).view(B, H, T, top).to(torch.int32)
    got = paged_block_attention(q.to(device), cache, pt, lt, cb.to(device), blocks.to(device), user_id=uid)
    k, v = P.keys_values(*parts, cb, uid)
    want, bound = torch.empty(B, G * H, T, 128).double(), torch.empty(B, G * H, T, 128).double()
    for b in range(B):
        for h in range(H):
            for t in range(T):
                seen = torch.zeros(n, page, dtype=torch.bool)
                seen[blocks[b, h, t].long()] = True
                seen = seen.view(-1)[:L]
                seen[L - T + t + 1:] = False
                o, e = P.attend(q[b, h * G:(h + 1) * G, t].double(), k[b, h][seen], v[b, h][seen],
                                torch.ones(G, int(seen.sum()), dtype=torch.bool), 1 / math.sqrt(128), dtype, False)
                want[b, h * G:(h + 1) * G, t], bound[b, h * G:(h + 1) * G, t] = o, e
    P.close(got, want, bound)


def _whole(x, dims):
    """int8 of x by the power of two that brings its largest (over `dims`) into [64, 128)."""
    most = x.abs().amax(dims, keepdim=True)
    e = torch.frexp(most)[1]
    return torch.where(most > 0, torch.round(torch.ldexp(x, 7 - e)).clamp(-127, 127), 0.0)


@pytest.mark.parametrize("B,H,G,T,n", [(1, 5, 3, 2, 2000), (2, 16, 2, 1, 1500), (1, 4, 9, 3, 9001), (1, 2, 4, 1, 20011), (1, 3, 2, 44, 17001)])
def test_selection_paths(device, B, H, G, T, n):
    """Scores ahead of the choice (few rows, many blocks) with kv heads of every kind, and rows that fill the chip with more
    blocks than LDS holds."""
    from omnistack_rs.cache import PagedKVCache, select_blocks
    page = 16
    cache = PagedKVCache(B * n, H, page, device=device, bounds=True)
    g = torch.Generator().manual_seed(331)
    c = torch.sort(torch.randint(0, 16, (2, B * n, H, 128), generator=g, dtype=torch.uint8), 0)[0]
    cache.k_bounds.copy_(c[0] | (c[1] << 4))
    pt = torch.randperm(B * n, generator=g).view(B, n)
    lens = torch.tensor([n * page - 7 - 900 * b for b in range(B)], dtype=torch.int32)
    q, cb = _q(B, G * H, T, 332, torch.bfloat16), P.codebooks(H)
    top, first, recent = 37, 2, 3
    got = select_blocks(q.to(device), cache, pt.to(torch.int32).to(device), lens.to(device), cb.to(device), top, first=first,
                        recent=recent, validate=False).cpu()
    cw = _whole(cb.double(), (1,))
    for b in range(B):
        x = q[b].double().view(H, G, T, 128)
        Q = _whole(torch.stack((x.clamp_min(0).sum(1), x.clamp_max(0).sum(1)), 2), (2, 3))         # (H, T, 2, 128)
        for h in range(H):
            hi, lo = cw[h][c[1, pt[b], h].long()], cw[h][c[0, pt[b], h].long()]                    # (n, 128)
            s = Q[h, :, 0] @ hi.T + Q[h, :, 1] @ lo.T                                              # whole numbers: exact
            for t in range(T):
                m = (int(lens[b]) - T + t + 1 + page - 1) // page
                st = s[t, :m].clone()
                st[:first] = st[m - recent:] = 1 << 40
                pick = torch.sort(torch.sort(st, descending=True, stable=True)[1][:top])[0]
                assert torch.equal(got[b, h, t].long(), pick), (b, h, t)


def test_pools_past_four_gigabytes(device):
    """Pages whose codes and bounds lie past 2^32 bytes give the bits of a small pool's."""
    from omnistack_rs.cache import PagedBlockAttention, PagedKVCache, paged_tree_attention, tree_masks
    H, page, L, Hq, T = 8, 16, 1000, 32, 3
    parts, cb = P.packed(1, H, L, seed=341), P.codebooks(H).to(device)
    small, pt, lt = P.paged(device, parts, page, spare=0, bounds=True)
    n = (1 << 22) + 200
    free, _ = torch.cuda.mem_get_info(device)
    if free < n * H * (page * 140 + 128) + (8 << 30):
        pytest.skip("needs 85 GB of free memory")
    big = PagedKVCache(n, H, page, device=device, bounds=True)
    ids = [n - 1 - 3 * i for i in range(small.n_pages)]
    for i, j in enumerate(ids):
        for name in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles"):
            getattr(big, name)[j].copy_(getattr(small, name)[i])
    far = torch.tensor(ids, dtype=torch.int32, device=device)[pt.long()]
    big.update_bounds(far, torch.zeros_like(lt), lt)
    assert all(torch.equal(big.k_bounds[j], small.k_bounds[i]) for i, j in enumerate(ids))
    q, tree = _q(1, Hq, T, 342, torch.bfloat16).to(device), tree_masks(torch.tensor([-1, 0, 0])).to(device)
    assert torch.equal(paged_tree_attention(q, big, far, lt, cb, tree), paged_tree_attention(q, small, pt, lt, cb, tree))
    a, b = (PagedBlockAttention(c, cb, Hq, 1, pt.shape[1], 9, T) for c in (big, small))
    assert torch.equal(a.run(q, far, lt), b.run(q, pt, lt)) and torch.equal(a.blocks, b.blocks)
    kept, at = torch.tensor([[2, 0]], dtype=torch.int32, device=device), lt - 3
    for c, table in ((big, far), (small, pt)):
        c.keep(table, at, kept)
    for i, j in enumerate(ids):
        for name in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles", "k_bounds"):
            assert torch.equal(getattr(big, name)[j], getattr(small, name)[i])


def test_prepared_objects_overlap(device):
    """Objects of their own on two streams, eager and as two graphs replayed at once, with splits, merges and scores ahead."""
    from omnistack_rs.cache import PagedBlockAttention, PagedTreeAttention, tree_masks
    B, Hq, H, L, page, T = 2, 16, 4, 24000, 16, 5
    parts, cb = P.packed(B, H, L, seed=351), P.codebooks(H).to(device)
    cache, pt, lt = P.paged(device, parts, page, bounds=True)
    tree = tree_masks(P.random_parents(B, T, 352)).to(device)
    calls = []
    for i in range(2):
        qt, qb = _q(B, Hq, T, 353 + i, torch.bfloat16).to(device), _q(B, Hq, 1, 355 + i, torch.bfloat16).to(device)
        tr, bl = PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], T), PagedBlockAttention(cache, cb, Hq, B, pt.shape[1], 60)
        assert tr.ws_bytes > 0 and bl.ws_bytes > 0
        calls.append((lambda tr=tr, qt=qt: tr.run(qt, pt, lt, tree)))
        calls.append((lambda bl=bl, qb=qb: bl.run(qb, pt, lt)))
    alone = [c().clone() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    graphs = []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c()
    for k in range(3):
        outs = []
        for c, s in zip(calls, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(o, a) for o, a in zip(outs, alone)), f"eager {k}"
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, a) for o, a in zip(outs, alone)), f"replay {k}"


def test_keep_of_nothing_narrows_the_bounds(device):
    """Where no drafted token is kept, the page of the last token that stays is that token's again."""
    from omnistack_rs.cache import PagedKVCache
    from omnistack_rs.kernels.quantize import PackedKVEncoder
    B, H, page = 2, 3, 16
    enc = PackedKVEncoder(P.codebooks(H).to(device), H, dtype=torch.float16, device=device)
    cache = PagedKVCache(8, H, page, device=device, bounds=True)
    pt = cache.page_table([cache.allocate(4 * page) for _ in range(B)])
    g = torch.Generator().manual_seed(361)
    at = torch.tensor([0, 0], dtype=torch.int32, device=device)
    k = torch.randn(B, H, 21, 128, generator=g).half().to(device)
    cache.append(enc, k, k, pt, at)
    before = cache.k_bounds[pt[:, :2].long()].clone()
    at = at + 21
    draft = 9 * torch.randn(B, H, 6, 128, generator=g).half().to(device)
    cache.append(enc, draft, draft, pt, at)
    assert not torch.equal(cache.k_bounds[pt[:, :2].long()], before)
    cache.keep(pt, at, torch.empty(B, 0, dtype=torch.int32, device=device))
    assert torch.equal(cache.k_bounds[pt[:, :2].long()], before)
    cache.append(enc, draft, draft, pt, at)
    cache.keep(pt, at, torch.full((B, 4), -1, dtype=torch.int32, device=device))
    assert torch.equal(cache.k_bounds[pt[:, :2].long()], before)


@pytest.mark.parametrize("B,H,G,T,L", [(1, 1, 1024, 2, 45), (2, 4096, 1, 1, 20), (1, 1, 200, 64, 70)])
def test_largest_groups_and_heads(device, B, H, G, T, L):
    """1024 query heads a kv head, 4096 kv heads, 12,800 rows a list."""
    from omnistack_rs.cache import PagedBlockAttention, paged_tree_attention, tree_masks
    lens = [L - 3 * b for b in range(B)]
    parts, cb = P.packed(B, H, L, seed=381), P.codebooks(H)
    q, tree = _q(B, G * H, T, 382, torch.bfloat16), tree_masks(P.random_parents(B, T, 383))
    cache, pt, lt = P.paged(device, parts, 16, lens, bounds=True)
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), tree.to(device), user_id=2, with_qjl=False)
    want, bound = _tree_want(q, parts, cb, 2, lens, tree, False)
    P.close(got, want, bound)
    # all of a sequence's blocks, for its last token: a chain's last row
    att = PagedBlockAttention(cache, cb.to(device), G * H, B, pt.shape[1], pt.shape[1], user_id=2, with_qjl=False)
    last = q[:, :, -1:].contiguous()
    w, e = _tree_want(last, parts, cb, 2, lens, torch.ones(B, 1, dtype=torch.int64), False)
    P.close(att.run(last.to(device), pt, lt), w, e)


def test_no_sequences(device):
    from omnistack_rs.cache import PagedBlockAttention, PagedTreeAttention
    parts, cb = P.packed(1, 2, 20, seed=391), P.codebooks(2).to(device)
    cache, pt, lt = P.paged(device, parts, 16, bounds=True)
    q = torch.empty(0, 8, 3, 128, dtype=torch.bfloat16, device=device)
    pt0, lt0, tree = pt[:0].contiguous(), lt[:0].contiguous(), torch.ones(3, dtype=torch.int64, device=device)
    assert PagedTreeAttention(cache, cb, 8, 0, pt.shape[1], 3).run(q, pt0, lt0, tree).shape == (0, 8, 3, 128)
    assert PagedBlockAttention(cache, cb, 8, 0, pt.shape[1], 2, 3).run(q, pt0, lt0).shape == (0, 8, 3, 128)
    cache.keep(pt0, lt0, torch.empty(0, 3, dtype=torch.int32, device=device))
    cache.update_bounds(pt0, lt0, lt0)
