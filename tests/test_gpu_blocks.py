"""Selection of each query's blocks by their keys' bounds (omni_block_bounds,
omni_block_select) and the attention over them (omni_attn_blocks), against
whole-number and 64-bit forms."""
import math

import pytest
import torch

from tests import _pages as P

pytestmark = pytest.mark.gpu


def _q(B, Hq, T, seed, dtype, size=1.0):
    return (size * torch.randn(B, Hq, T, 128, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _bounds(kn, L, page):
    """(H, blocks, 128) least and largest codes of one sequence's blocks, kn (H, S, 64)."""
    c = P.codes(kn[:, :L])
    cut = [c[:, i:i + page] for i in range(0, L, page)]
    return torch.stack([x.amin(1) for x in cut], 1), torch.stack([x.amax(1) for x in cut], 1)


def _whole(x):
    most = float(x.abs().max())
    return torch.round(x * 2.0 ** (7 - math.frexp(most)[1])).clamp(-127, 127).long() if most > 0 else torch.zeros_like(x).long()


def _select(q, kn, cb, lens, page, top, first, recent, flip, rotate):
    """(B, H, T, top) by Python's exact arithmetic on the definition."""
    B, Hq, T, _ = q.shape
    H = kn.shape[1]
    G = Hq // H
    x = q.double() if not rotate else P.rotated(q, flip) * math.sqrt(128.0)
    if rotate:                                       # unnormalized sums of 16-bit values: exact without the factor
        i = torch.arange(128)
        odd = sum(((i[:, None] & i[None, :]) >> b) & 1 for b in range(7)) % 2
        x = (q.double() if flip is None else q.double() * flip.double()) @ (1.0 - 2.0 * odd.double())
    out = torch.full((B, H, T, top), -1, dtype=torch.int32)
    scores = {}
    for b in range(B):
        if lens[b] == 0:
            continue
        lo, hi = _bounds(kn[b], lens[b], page)
        for t in range(T):
            seen = lens[b] - T + 1 + t
            if seen <= 0:
                continue
            n = (seen + page - 1) // page
            for h in range(H):
                rows = x[b, h * G:(h + 1) * G, t]
                Q = _whole(torch.stack((rows.clamp_min(0).sum(0), rows.clamp_max(0).sum(0))))
                c = _whole((cb[h] if cb.dim() == 2 else cb).double())
                s = (c[hi[h, :n]] * Q[0]).sum(1) + (c[lo[h, :n]] * Q[1]).sum(1)
                s = s.tolist()
                scores[b, h, t] = s
                edge = set(range(min(first, n))) | set(range(max(0, n - recent), n))
                order = sorted(range(n), key=lambda j: (j not in edge, -s[j], j))
                pick = sorted(order[:top])
                out[b, h, t, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out, scores


def _attend(q, parts, cb, uid, lens, page, blocks, with_qjl, rotate, flip, scale):
    B, Hq, T, _ = q.shape
    k, v = P.keys_values(*parts, cb, uid, with_qjl)
    G = Hq // k.shape[1]
    x = P.rotated(q, flip) if rotate else q.double()
    want = torch.full((B, Hq, T, 128), float("nan")).double()
    bound = torch.zeros_like(want)
    for b in range(B):
        for t in range(T):
            seen = lens[b] - T + 1 + t
            for h in range(Hq):
                tok = [j * page + i for j in blocks[b, h // G, t].tolist() if j >= 0 for i in range(page) if j * page + i < seen]
                if tok:
                    o, e = P.attend(x[b, h, t][None], k[b, h // G, tok], v[b, h // G, tok],
                                    torch.ones(1, len(tok), dtype=torch.bool), scale, q.dtype, rotate)
                    want[b, h, t], bound[b, h, t] = o[0], e[0]
    return want, bound


CASES = [
    # B, Hq, H, T, lens, page, top, first, recent, dtype, qjl, rotate
    (2, 8, 2, 1, [1, 16], 16, 2, 1, 1, torch.bfloat16, True, False),
    (3, 8, 2, 1, [600, 33, 17], 16, 4, 1, 1, torch.bfloat16, True, True),
    (2, 8, 8, 3, [2, 1001], 32, 7, 0, 2, torch.float16, True, False),
    (1, 10, 2, 5, [2049], 64, 9, 2, 3, torch.bfloat16, False, True),
    (1, 7, 1, 1, [9000], 16, 40, 1, 1, torch.float16, True, True),
    (2, 40, 2, 2, [700, 1500], 128, 2, 1, 1, torch.bfloat16, True, False),      # 20 heads a group; the edges alone
    (1, 4, 4, 1, [5000], 1024, 3, 0, 1, torch.bfloat16, True, False),
    (1, 2, 1, 1, [40000], 16, 300, 3, 5, torch.bfloat16, True, True),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_selection_and_attention(device, case):
    from omnistack_rs.cache import PagedBlockAttention, paged_block_attention, select_blocks
    B, Hq, H, T, lens, page, top, first, recent, dtype, qjl, rotate = case
    uid = 6
    parts, cb = P.packed(B, H, max(lens), seed=171), P.codebooks(H)
    q = _q(B, Hq, T, 172, dtype)
    flip = (torch.randint(0, 2, (128,), generator=torch.Generator().manual_seed(4)) * 2 - 1).to(torch.int8)
    cache, pt, lt = P.paged(device, parts, page, lens, seed=page, bounds=True)
    for b in range(B):
        lo, hi = _bounds(parts[0][b], lens[b], page)
        n = lo.shape[1]
        assert torch.equal(cache.k_bounds[pt[b, :n].long()].cpu().long().transpose(0, 1), lo | (hi << 4))
    sel = dict(first=first, recent=recent, rotate_q=rotate, sign_flip=flip.to(device))
    got = select_blocks(q.to(device), cache, pt, lt, cb.to(device), top, **sel)
    want, _ = _select(q, parts[0], cb, lens, page, top, first, recent, flip, rotate)
    assert torch.equal(got.cpu(), want)
    kw = dict(user_id=uid, with_qjl=qjl, rotate_q=rotate, sign_flip=flip.to(device))
    o = paged_block_attention(q.to(device), cache, pt, lt, cb.to(device), got, **kw)
    w, e = _attend(q, parts, cb, uid, lens, page, want, qjl, rotate, flip, 1 / math.sqrt(128))
    assert o.dtype == dtype
    P.close(o, w, e, str(case))
    # the order of the blocks, and numbers outside the query's, do not matter
    mixed = torch.cat((got.flip(-1), torch.full_like(got[..., :1], 1 << 30), torch.full_like(got[..., :1], -7)), -1)
    P.close(paged_block_attention(q.to(device), cache, pt, lt, cb.to(device), mixed, **kw), w, e, f"mixed {case}")
    wide = torch.full((B, pt.shape[1] + 30), -1, dtype=torch.int32, device=device)
    wide[:, :pt.shape[1]] = pt
    att = PagedBlockAttention(cache, cb.to(device), Hq, B, wide.shape[1], top, T, first, recent, q_dtype=dtype, **kw)
    P.close(att.run(q.to(device), wide, lt), w, e, f"prepared {case}")
    assert torch.equal(att.blocks.cpu(), want)


def test_bound_holds(device):
    """The score is no less than any key's own, up to the whole numbers' rounding (half a step of 1/64 of the largest, per
    dim and factor)."""
    B, Hq, H, T, L, page = 1, 8, 2, 1, 500, 16
    parts, cb = P.packed(B, H, L, seed=181), P.codebooks(H)
    q = _q(B, Hq, T, 182, torch.float16)
    _, scores = _select(q, parts[0], cb, [L], page, 40, 1, 1, None, False)
    k, _ = P.keys_values(*parts, cb, 0, False)
    for h in range(H):
        rows = q[0, h * 4:(h + 1) * 4, 0].double()
        Q = torch.stack((rows.clamp_min(0).sum(0), rows.clamp_max(0).sum(0)))
        sq, sc = 2.0 ** (7 - math.frexp(float(Q.abs().max()))[1]), 2.0 ** (7 - math.frexp(float(cb[h].abs().max()))[1])
        own = (rows @ k[0, h].T).sum(0) * sq * sc
        # each of 256 terms: at most 128 of one factor times half a step of the other, and a quarter (or a clamp of one)
        slack = 256 * (128 + 128 + 1)
        for j, s in enumerate(scores[0, h, 0]):
            assert s + slack >= float(own[j * page:(j + 1) * page].max())


def test_ties_go_to_the_lowest(device):
    """Equal pages have equal scores; the first of them are taken."""
    from omnistack_rs.cache import select_blocks
    B, Hq, H, page, n = 1, 8, 2, 16, 900
    parts = list(P.packed(B, H, page, seed=191))
    parts = [t.repeat(1, 1, n, *([1] * (t.dim() - 3))) for t in parts]
    cache, pt, lt = P.paged(device, parts, page, bounds=True)
    cb, q = P.codebooks(H).to(device), _q(B, Hq, 1, 192, torch.bfloat16).to(device)
    got = select_blocks(q, cache, pt, lt, cb, 10, first=2, recent=3)
    assert got.cpu()[0, :, 0].tolist() == [[0, 1, 2, 3, 4, 5, 6, n - 3, n - 2, n - 1]] * H
    # a page whose codes reach further in every dim stands above all of them
    cache.k_bounds[pt[0, 500].long()] = 0xF0
    got = select_blocks(q, cache, pt, lt, cb, 6, first=0, recent=1)
    assert got.cpu()[0, :, 0].tolist() == [[0, 1, 2, 3, 500, n - 1]] * H
    # a query of zeros knows no difference
    got = select_blocks(torch.zeros_like(q), cache, pt, lt, cb, 4)
    assert got.cpu()[0, :, 0].tolist() == [[0, 1, 2, n - 1]] * H


def test_many_blocks(device):
    """More blocks than the selection holds in LDS, scores of every size."""
    from omnistack_rs.cache import PagedKVCache, select_blocks
    H, page, n = 2, 16, 30011
    cache = PagedKVCache(n, H, page, device=device, bounds=True)
    g = torch.Generator().manual_seed(7)
    c = torch.sort(torch.randint(0, 16, (2, n, H, 128), generator=g), 0)[0]
    few = torch.rand(n, generator=g) < 0.5                      # half of the pages from a handful of patterns
    c[:, few] = c[:, torch.randint(0, 5, (int(few.sum()),), generator=g)]
    cache.k_bounds.copy_((c[0] | (c[1] << 4)).to(torch.uint8))
    order = torch.randperm(n, generator=g)
    pt = order[None].to(torch.int32).to(device)
    q, cb = _q(1, 4, 1, 202, torch.bfloat16), P.codebooks(H)
    Lt = torch.tensor([n * page - 3], dtype=torch.int32, device=device)
    for top in (2, 3, 100, 5000, n - 1):
        got = select_blocks(q.to(device), cache, pt, Lt, cb.to(device), top, validate=False).cpu()
        for h in range(H):
            rows = q[0, h * 2:(h + 1) * 2, 0].double()
            Q = _whole(torch.stack((rows.clamp_min(0).sum(0), rows.clamp_max(0).sum(0))))
            cw = _whole(cb[h].double())
            s = ((cw[c[1, order, h]] * Q[0]).sum(1) + (cw[c[0, order, h]] * Q[1]).sum(1))
            s[0] = s[n - 1] = 1 << 40
            pick = torch.sort(torch.sort(s, descending=True, stable=True)[1][:top])[0]
            assert torch.equal(got[0, h, 0].long(), pick), (top, h)


def test_rows_without_tokens_bad_pages_and_lengths(device):
    from omnistack_rs.cache import paged_block_attention, select_blocks
    B, Hq, H, T, page = 5, 8, 2, 2, 16
    lens = [0, 1, 200, 300, 90]
    parts, cb, q = P.packed(B, H, 300, seed=211), P.codebooks(H).to(device), _q(B, Hq, T, 212, torch.bfloat16).to(device)
    cache, pt, lt = P.paged(device, parts, page, lens, bounds=True)
    pt[3, 7] = cache.n_pages + 5
    lt[4] = pt.shape[1] * page + 1
    with pytest.raises((ValueError, IndexError)):
        select_blocks(q, cache, pt, lt, cb, 4)
    got = select_blocks(q, cache, pt, lt, cb, 4, validate=False)
    assert (got[0] == -1).all() and (got[1, :, 0] == -1).all() and got[1, :, 1].tolist() == [[0, -1, -1, -1]] * H
    assert (got[4] == -1).all()
    assert (got[3] == 7).any(-1).all()                       # the bad page is selected, and so is seen
    o = paged_block_attention(q, cache, pt, lt, cb, got, validate=False)
    assert torch.isnan(o[0]).all() and torch.isnan(o[1, :, 0]).all() and torch.isfinite(o[1, :, 1]).all()
    assert torch.isfinite(o[2]).all() and torch.isnan(o[3:]).all()


def test_hidden_tokens_reach_nobody(device):
    """What lies in blocks that are not selected, and behind a query's last token
    within a selected one, leaves its bits alone."""
    from omnistack_rs.cache import paged_block_attention
    B, Hq, H, T, L, page = 1, 8, 2, 3, 75, 32
    parts, cb = P.packed(B, H, L, seed=221), P.codebooks(H).to(device)
    q = _q(B, Hq, T, 222, torch.float16).to(device)
    cache, pt, lt = P.paged(device, parts, page)
    blocks = torch.tensor([[0, 2, -1]], dtype=torch.int32, device=device).expand(B, H, T, 3).contiguous()
    ref = paged_block_attention(q, cache, pt, lt, cb, blocks)
    cache.k_norms[pt[0, 1].long()] = float("nan")
    cache.v_nibbles[pt[0, 1].long()] ^= 0x3C
    assert torch.equal(paged_block_attention(q, cache, pt, lt, cb, blocks), ref)
    cache.k_norms[pt[0, 2].long(), :, (L - 1) % page:] = float("nan")      # the last token, which the last query alone sees
    got = paged_block_attention(q, cache, pt, lt, cb, blocks)
    assert torch.equal(got[:, :, :2], ref[:, :, :2]) and torch.isnan(got[:, :, 2]).all()


def test_all_blocks_equal_a_tree_of_one(device):
    from omnistack_rs.cache import PagedBlockAttention, paged_tree_attention
    B, Hq, H, L, page = 2, 8, 2, 777, 16
    parts, cb = P.packed(B, H, L, seed=231), P.codebooks(H).to(device)
    q = _q(B, Hq, 1, 232, torch.bfloat16).to(device)
    cache, pt, lt = P.paged(device, parts, page, bounds=True)
    att = PagedBlockAttention(cache, cb, Hq, B, pt.shape[1], pt.shape[1], user_id=2)
    ref = paged_tree_attention(q, cache, pt, lt, cb, torch.ones(1, dtype=torch.int64, device=device), user_id=2)
    assert torch.equal(att.run(q, pt, lt), ref)               # the same tiles in the same waves


def test_bounds_follow_appends_and_writes(device):
    from omnistack_rs.cache import PagedKVCache
    from omnistack_rs.kernels.quantize import PackedKVEncoder
    B, H, page = 3, 5, 32
    enc = PackedKVEncoder(P.codebooks(H).to(device), H, dtype=torch.float16, device=device)
    cache = PagedKVCache(24, H, page, device=device, bounds=True)
    cache.k_bounds.fill_(0x77)
    pt = cache.page_table([cache.allocate(6 * page) for _ in range(B)])
    g = torch.Generator().manual_seed(9)
    pos = torch.tensor([0, 31, 70], dtype=torch.int32, device=device)
    for T in (50, 1, 1, 33):
        k = torch.randn(B, H, T, 128, generator=g).half().to(device)
        cache.append(enc, k, k, pt, pos)
        for b in range(B):
            for p in range(int(pos[b]) // page, (int(pos[b]) + T - 1) // page + 1):
                n, i = min(page, int(pos[b]) + T - p * page), int(pt[b, p])
                c = P.codes(cache.k_nibbles[i, :, :n].cpu())
                assert torch.equal(cache.k_bounds[i].cpu().long(), c.amin(1) | (c.amax(1) << 4)), (T, b, p)
        pos = pos + T
    used = set(pt.flatten().tolist())
    rest = [i for i in range(cache.n_pages) if i not in used]
    assert (cache.k_bounds[rest] == 0x77).all()
    # positions outside the table, pages outside the pool
    before = cache.k_bounds.clone()
    pt2 = pt.clone()
    pt2[0] = -1
    pt2[1] = cache.n_pages
    cache.update_bounds(pt2, torch.tensor([0, 0, 300], dtype=torch.int32, device=device),
                        torch.tensor([90, 90, 400], dtype=torch.int32, device=device))
    assert torch.equal(cache.k_bounds, before)


def test_capture_and_streams(device):
    from omnistack_rs.cache import PagedBlockAttention
    B, Hq, H, L, page, top = 3, 16, 4, 5000, 16, 20
    parts, cb = P.packed(B, H, L, seed=241), P.codebooks(H).to(device)
    cache, pt, lt = P.paged(device, parts, page, bounds=True)
    att, ref = (PagedBlockAttention(cache, cb, Hq, B, pt.shape[1], top) for _ in range(2))
    qs, ls = _q(B, Hq, 1, 242, torch.bfloat16).to(device), lt.clone()
    att.run(qs, pt, ls)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = att.run(qs, pt, ls)
    side = torch.cuda.Stream()
    for k in range(4):
        qs.copy_(_q(B, Hq, 1, 250 + k, torch.bfloat16))
        ls.copy_(lt - 700 * k)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = ref.run(qs, pt, ls)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(att.blocks, ref.blocks), f"replay {k}"
        torch.zeros(1 << 20, device=device).sum().item()


def test_refusals(device):
    from omnistack_rs.cache import PagedBlockAttention, paged_block_attention, select_blocks
    B, Hq, H, T, page = 2, 8, 2, 1, 16
    parts, cb = P.packed(B, H, 100, seed=251), P.codebooks(H).to(device)
    cache, pt, lt = P.paged(device, parts, page, bounds=True)
    plain, _, _ = P.paged(device, parts, page)
    q = _q(B, Hq, T, 252, torch.bfloat16).to(device)
    blocks = select_blocks(q, cache, pt, lt, cb, 4)
    for args, kw in (((q, plain, pt, lt, cb, 4), {}), ((q, cache, pt, lt, cb, 1), {}), ((q, cache, pt, lt, cb, 4), dict(recent=0)),
                     ((q, cache, pt, lt, cb, 4), dict(first=-1)), ((q, cache, pt, lt, cb.flip(1), 4), {}),
                     ((q.float(), cache, pt, lt, cb, 4), {}), ((q, cache, pt[:1], lt, cb, 4), {})):
        with pytest.raises(ValueError):
            select_blocks(*args, **kw)
    twice = blocks.clone()
    twice[..., 1] = twice[..., 0]
    for bad in (blocks.long(), blocks[:1], blocks[:, :1], blocks[..., :0], twice):
        with pytest.raises(ValueError):
            paged_block_attention(q, cache, pt, lt, cb, bad)
    for kw in (dict(scale=-1.0), dict(scale=0.0), dict(top=1), dict(first=4)):
        with pytest.raises(ValueError):
            PagedBlockAttention(cache, cb, Hq, B, pt.shape[1], **{"top": 4, **kw})
    with pytest.raises(ValueError):
        PagedBlockAttention(plain, cb, Hq, B, pt.shape[1], 4)
    with pytest.raises(ValueError):
        PagedBlockAttention(cache, cb.flip(1), Hq, B, pt.shape[1], 4)
    with pytest.raises(ValueError):
        plain.update_bounds(pt, lt, lt)
    assert select_blocks(q[:0], cache, pt[:0], lt[:0], cb, 4).shape == (0, H, T, 4)
