"""The bounds of the pages' key codes where tokens are written out of order, moved
and dropped, and in tables of every width."""
import math

import pytest
import torch

from tests import _pages as P

pytestmark = pytest.mark.gpu


def _want(cache, page, n):
    """The bounds of a page's first n tokens, from the pool's codes."""
    c = P.codes(cache.k_nibbles[page, :, :n].cpu())
    return c.amin(1) | (c.amax(1) << 4)


def _put(cache, pages, parts, a, b, **kw):
    cache.write(pages, *(t[0, :, a:b] for t in parts), start=a, **kw)


def test_writes_before_a_sequence_s_end(device):
    """The front of a sequence written again, and pieces out of order, with the sequence's length: every token counts."""
    from omnistack_rs.cache import PagedKVCache
    H, ps, S = 3, 16, 45
    parts = P.packed(1, H, S, seed=501)
    cache = PagedKVCache(5, H, ps, device=device, bounds=True)
    pages = cache.allocate(S)
    lens = (16, 16, 13)

    def check():
        for p, n in zip(pages, lens):
            assert torch.equal(cache.k_bounds[p].cpu().long(), _want(cache, p, n)), p

    _put(cache, pages, parts, 0, S)
    check()
    narrow = list(P.packed(1, H, S, seed=502))
    narrow[0] = torch.full_like(narrow[0], 0x88)                       # a code in the middle: later tokens alone reach further
    _put(cache, pages, narrow, 0, 4, length=S)
    check()
    assert not torch.equal(cache.k_bounds[pages[0]].cpu().long(), _want(cache, pages[0], 4))
    _put(cache, pages, narrow, 33, 36, length=S)
    check()
    cache.k_nibbles.zero_()
    cache.k_bounds.zero_()
    for a, b in ((40, 45), (20, 37), (8, 20), (37, 40), (0, 8)):       # each piece once, in no order
        _put(cache, pages, parts, a, b, length=S)
    check()
    _put(cache, pages, parts, 0, 20)                                   # no length: the sequence ends here
    assert torch.equal(cache.k_bounds[pages[1]].cpu().long(), _want(cache, pages[1], 4))
    for kw in (dict(length=19), dict(length=49), dict(length=-1)):
        before = cache.k_nibbles.clone()
        with pytest.raises(ValueError):
            _put(cache, pages, narrow, 0, 20, **kw)
        assert torch.equal(cache.k_nibbles, before)


def test_kept_numbers_outside_the_tree(device):
    """Entries that keep() passes over, 64 and above among them, put no token into the bounds."""
    from omnistack_rs.cache import PagedKVCache
    H, ps, L = 3, 16, 10
    parts = P.packed(2, H, L + 5, seed=511)
    caches = []
    for last in (70, -1, 64, 1 << 30, -(1 << 31)):
        cache = PagedKVCache(4, H, ps, device=device, bounds=True)
        pages = [cache.allocate(L + 5) for _ in range(2)]
        for b in range(2):
            cache.write(pages[b], *(t[b] for t in parts))
        kept = torch.tensor([[3, last, -1], [last, last, last]], dtype=torch.int32, device=device)
        cache.keep(cache.page_table(pages), torch.full((2,), L, dtype=torch.int32, device=device), kept, validate=False)
        for b, n in ((0, L + 1), (1, L)):
            assert torch.equal(cache.k_bounds[pages[b][0]].cpu().long(), _want(cache, pages[b][0], n)), (last, b)
        caches.append(cache)
    for c in caches[1:]:
        for name in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles", "k_bounds"):
            assert torch.equal(getattr(c, name), getattr(caches[0], name)), name


def test_tables_of_more_pages_than_a_grid_holds(device):
    """A sequence over 2^24 pages, most of them outside the pool; any count of tokens."""
    from omnistack_rs import _lib
    from omnistack_rs.cache import PagedKVCache
    H, ps, n = 2, 16, (1 << 24) + 40
    cache = PagedKVCache(6, H, ps, device=device, bounds=True)
    cache.k_nibbles.random_(0, 256, generator=torch.Generator(device=device).manual_seed(521))
    table = torch.full((1, n), -1, dtype=torch.int32, device=device)
    where = {1: 0, 2: 1 << 20, 3: (1 << 24) - 1, 4: (1 << 24) + 3}            # page: its place
    for page, i in where.items():
        table[0, i] = page
    end = where[4] * ps + 5
    ends = torch.tensor([end], dtype=torch.int32, device=device)

    def check():
        for page in range(6):
            want = _want(cache, page, 5 if page == 4 else ps) if page in where else torch.zeros(H, 128).long()
            assert torch.equal(cache.k_bounds[page].cpu().long(), want), page

    cache.update_bounds(table, torch.zeros_like(ends), ends)
    check()
    L = _lib.lib()
    for start, count in ((0, end), (-9, end + 9)):
        cache.k_bounds.zero_()
        cache._bounds(table, torch.tensor([start], dtype=torch.int32, device=device), None, count)
        check()
    # counts far past the table's end: every page whole
    for count in (1 << 31, (1 << 62) + 3, (1 << 63) - 1):
        cache.k_bounds.zero_()
        starts = torch.tensor([0], dtype=torch.int32, device=device)
        assert L.omni_block_bounds(cache.k_nibbles.data_ptr(), cache.k_bounds.data_ptr(), 6, H, ps, table.data_ptr(), n,
                                   starts.data_ptr(), None, count, 1, _lib.stream_of(device)) == 0
        assert torch.equal(cache.k_bounds[4].cpu().long(), _want(cache, 4, ps)) and torch.equal(
            cache.k_bounds[1].cpu().long(), _want(cache, 1, ps))


def _scaled(x):
    """x by the power of two that brings its largest into [64, 128), and rounded to whole numbers."""
    x = x * 2.0 ** (7 - math.frexp(float(x.abs().max()))[1])
    return x, torch.round(x).clamp(-127, 127)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [1, 4])
def test_selected_blocks_bound_the_others_keys(device, G, dtype):
    """No key of a block that was passed over scores above the bound of one that was taken, by more than the whole numbers'
    rounding: of this query and codebook, the sum over dims of the largest difference that any code makes, for both."""
    from omnistack_rs.cache import select_blocks
    H, ps, n, top, first, recent = 2, 16, 700, 60, 2, 3
    g = torch.Generator().manual_seed(531)
    cb = P.codebooks(H)
    q = (torch.randn(1, H, 1, 1, 128, generator=g) + 0.2 * torch.randn(1, H, G, 1, 128, generator=g)).reshape(1, H * G, 1, 128).to(dtype)
    Q = q.double().view(H, G, 128)
    # in every page one token follows the query's signs in some dims, none to all, the rest keep to the codes around zero
    kc = torch.randint(6, 10, (H, n, ps, 128), generator=g)
    with_q = torch.rand(H, n, 128, generator=g) < torch.rand(1, n, 1, generator=g)
    best = torch.where(Q.sum(1) > 0, 15, 0)[:, None].expand(H, n, 128)
    at = torch.randint(0, ps, (n,), generator=g)
    kc[:, torch.arange(n), at] = torch.where(with_q, best, kc[:, torch.arange(n), at])
    kc = kc.view(1, H, n * ps, 128).to(torch.uint8)
    parts = P.packed(1, H, n * ps, seed=532)
    kn = kc[..., 0::2] | (kc[..., 1::2] << 4)
    cache, pt, lt = P.paged(device, (kn, *parts[1:]), ps, bounds=True)
    got = select_blocks(q.to(device), cache, pt, lt, cb.to(device), top, first=first, recent=recent).cpu()[0, :, 0].long()
    told_apart = 0
    for h in range(H):
        c = cb[h].double()
        parts_q = torch.stack((Q[h].clamp_min(0).sum(0), (-Q[h]).clamp_min(0).sum(0)))
        (sq, wq), (sc, wc) = _scaled(parts_q), _scaled(c)
        slack = float((sq[..., None] * sc - wq[..., None] * wc).abs().amax(-1).sum())
        unit = float((sq.sum() / parts_q.sum()) * (sc.abs().sum() / c.abs().sum()))          # the powers of two
        codes = kc[0, h].view(n, ps, 128).long()
        own = (c[codes] @ Q[h].sum(0)).amax(1) * unit                                       # a page's best key
        bound = (c[codes.amax(1)] @ parts_q[0] - c[codes.amin(1)] @ parts_q[1]) * unit
        assert bool((own <= bound + 1e-6).all())
        taken = torch.zeros(n, dtype=torch.bool)
        taken[got[h]] = True
        assert int(taken.sum()) == top and taken[:first].all() and taken[n - recent:].all()
        inner = torch.arange(n).ge(first) & torch.arange(n).lt(n - recent)
        least = float(bound[taken & inner].min())
        assert float(own[~taken].max()) <= least + 2 * slack
        told_apart += int((own[inner].max() > bound[inner] + 2 * slack).sum())
    assert told_apart > n // 2                                # most pages, if taken, would have failed


def test_a_drafting_step_captured(device):
    """Append, tree attention, keep and the attention over selected blocks as one graph, replayed over a growing cache, against
    the same step run eagerly on a cache of its own."""
    from omnistack_rs.cache import PagedBlockAttention, PagedKVCache, PagedTreeAttention, tree_masks
    from omnistack_rs.kernels.quantize import PackedKVEncoder
    B, Hq, H, T, ps, top, uid = 3, 8, 2, 6, 16, 5, 7
    cb = P.codebooks(H).to(device)
    enc = PackedKVEncoder(cb, H, user_id=uid, dtype=torch.bfloat16, device=device)
    g = torch.Generator().manual_seed(541)
    tree = tree_masks(torch.tensor([-1, 0, 0, 1, 2, 3])).to(device)
    first = torch.randn(B, H, 90, 128, generator=g).to(torch.bfloat16).to(device)
    sides = []
    for _ in range(2):
        cache = PagedKVCache(60, H, ps, device=device, bounds=True)
        pt = cache.page_table([cache.allocate(300) for _ in range(B)])
        cache.append(enc, first, first, pt, torch.zeros(B, dtype=torch.int32, device=device))
        att = PagedTreeAttention(cache, cb, Hq, B, pt.shape[1], T, user_id=uid)
        sparse = PagedBlockAttention(cache, cb, Hq, B, pt.shape[1], top, user_id=uid)
        sides.append((cache, pt, att, sparse))
    k, v = (torch.zeros(B, H, T, 128, dtype=torch.bfloat16, device=device) for _ in range(2))
    q, q1 = (torch.zeros(B, Hq, t, 128, dtype=torch.bfloat16, device=device) for t in (T, 1))
    kept = torch.full((B, 4), -1, dtype=torch.int32, device=device)
    lens = [torch.tensor([90, 80, 33], dtype=torch.int32, device=device) for _ in range(2)]

    def step(i):
        cache, pt, att, sparse = sides[i]
        cache.append(enc, k, v, pt, lens[i], validate=False)
        o = att.run(q, pt, lens[i] + T, tree)
        cache.keep(pt, lens[i], kept, validate=False)
        lens[i] += (kept >= 0).sum(1, dtype=torch.int32)
        return o, sparse.run(q1, pt, lens[i])

    step(1)                                                       # nothing kept: the lengths stay
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(1)
    for i, paths in enumerate(([[0, 1, 3], [0], []], [[], [0, 2, 4], [0, 1, 3, 5]], [[0, 2], [0, 1], [0]], [[0], [], [0, 1]])):
        for t in (k, v, q, q1):
            t.copy_(torch.randn(t.shape, generator=g))
        kept.fill_(-1)
        for b, p in enumerate(paths):
            kept[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        want = [t.clone() for t in step(0)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lens[0], lens[1]) and all(torch.equal(a, b) for a, b in zip(outs, want)), i
        assert torch.equal(sides[0][3].blocks, sides[1][3].blocks)
        for name in ("k_nibbles", "k_qjl", "k_norms", "v_nibbles", "k_bounds"):
            a, b = (getattr(s[0], name)[s[1].long()] for s in sides)
            assert torch.equal(a, b), (i, name)
        torch.zeros(1 << 20, device=device).sum().item()
