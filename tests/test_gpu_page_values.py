"""The attention over drafted tokens' trees and selected blocks where its
arithmetic could go wrong: one key far above a long tail, large scores, large
norms, sums that nearly cancel.  Results are known in closed form; each
tolerance is derived beside its use."""
import math

import pytest
import torch

from tests import _pages as P

pytestmark = pytest.mark.gpu

CB = P.codebooks(1)[0] / P.codebooks(1)[0, -1] * 2.7326            # N(0, 1)'s levels, ascending


def _pool(device, kc, vc, page, kr=None):
    """One head's tokens (codes kc, vc: (S, 128)) as a pool of one sequence."""
    kn, vn = (c[None, None, :, 0::2] | (c[None, None, :, 1::2] << 4) for c in (kc, vc))
    S = kc.shape[0]
    kq = torch.full((1, 1, S, 8), 0xFF, dtype=torch.uint8)
    kr = torch.zeros(1, 1, S) if kr is None else kr.view(1, 1, S)
    return P.paged(device, (kn, kq, kr, vn), page)


def _same(n, code):
    return torch.full((n, 128), code, dtype=torch.uint8)


def test_a_tail_far_below_one_key(device):
    """One key and 131071 others, each 2^-25.1 of it: together 3.6e-3.  More than
    four lists a compute unit, so that none is split: a wave's eighth of the tail
    is held against the key itself."""
    from omnistack_rs.cache import paged_tree_attention
    S, B = 131072, 1100
    kc, vc = _same(S, 8), _same(S, 0)
    kc[0], vc[0] = 15, 15
    cache, pt, lt = _pool(device, kc, vc, 1024)
    a = 25.1 * math.log(2) * math.sqrt(128) / (128 * float(CB[15] - CB[8]))
    q = torch.full((B, 1, 1, 128), a, dtype=torch.float16)
    got = paged_tree_attention(q.to(device), cache, pt.expand(B, -1).contiguous(), lt.expand(B).contiguous(), CB.to(device),
                               torch.ones(1, dtype=torch.int64, device=device), with_qjl=False, validate=False).double().cpu()
    gap = float(q[0, 0, 0, 0]) * 128 * (float(CB[15]) - float(CB[8])) / math.sqrt(128)
    assert 25.0 < gap / math.log(2) < 25.2
    w = (S - 1) * math.exp(-gap)
    want = float(CB[15]) * (1 - w) / (1 + w)
    # the output's half step; of the tail's weights the rounding of P, 2^-25 of 2^-18 or more, and of their scores, 2^-16
    # of 19; V's 22 bits
    off = 2.0 ** -11 * want + 2 * w * float(CB[15]) * (2.0 ** -7 + 2.0 ** -11) + 2.0 ** -20
    assert float((got - want).abs().max()) <= off


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1.5e7])
def test_large_scores(device, size, dtype):
    """The key of the largest score takes all, however large, of either sign, alone
    or among others; 64 rows whose scores' roundings differ."""
    from omnistack_rs.cache import paged_tree_attention
    S, T = 300, 64
    g = torch.Generator().manual_seed(5)
    kc, vc = _same(S, 8), torch.randint(0, 16, (S, 128), generator=g, dtype=torch.uint8)
    kc[77], kc[78] = 15, 0
    cache, pt, lt = _pool(device, kc, vc, 16)
    top = 128 * float(CB[15])
    q = ((0.7 + 0.3 * torch.rand(1, 1, T, 1, generator=g)) * torch.tensor([1.0, -1.0]).repeat(32)[None, None, :, None])
    q = q.expand(1, 1, T, 128).to(dtype).contiguous()
    none = torch.zeros(T, dtype=torch.int64, device=device)        # the cached tokens alone
    for n, first in ((S, 0), (1, 77), (1, 78)):                    # all; each of the two alone
        if n == S:
            c, table, lens = cache, pt, lt
        else:
            c, table, lens = _pool(device, kc[first:first + 1], vc[first:first + 1], 16)
        # T drafted tokens that nobody sees behind them
        more = torch.full((1, table.shape[1] + 4), int(table[0, 0]), dtype=torch.int32, device=device)
        more[0, :table.shape[1]] = table[0]
        got = paged_tree_attention(q.to(device), c, more, lens + T, CB.to(device), none, scale=size / top, with_qjl=False)
        for t in range(T):
            v = CB[vc[(77 if t % 2 == 0 else 78) if n == S else first].long()].double()
            # the output's half step, V's 22 bits; other keys: exp(-0.6 * 100) and less
            err = (got[0, 0, t].double().cpu() - v).abs()
            assert bool((err <= torch.finfo(dtype).eps / 2 * v.abs() + 2.0 ** -20).all()), (n, first, t)


@pytest.mark.parametrize("B,T,G", [(1, 2, 4), (1, 8, 4), (1, 12, 4), (1, 16, 4), (160, 8, 4), (3, 1, 40)])
@pytest.mark.parametrize("size", [4.0 * 65500, 4.0 * 65510, 1e7, 1e15, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_norms(device, size, dtype, B, T, G):
    """Residual norms around and far beyond 65504 of the power of two above the largest centroid (4), some tokens of a tile
    with one and some without, scores of a size that keeps every token's weight."""
    from omnistack_rs.cache import paged_block_attention, paged_tree_attention
    H, S, uid, page = 2, 45, 3, 16
    parts, cb = list(P.packed(1, H, S, seed=401)), CB.repeat(H, 1)
    for s, part in ((3, 1.0), (17, 0.5), (20, 0.9), (39, 0.25)):
        parts[2][:, :, s] = size * part
    cache, pt, lt = P.paged(device, parts, page)
    pt, lt = pt.expand(B, -1).contiguous(), lt.expand(B).contiguous()
    q = torch.randn(1, G * H, T, 128, generator=torch.Generator().manual_seed(402)).to(dtype)
    scale = 4.0 / size
    k, v = P.keys_values(*parts, cb, uid)
    args = (q.expand(B, -1, -1, -1).contiguous().to(device), cache, pt, lt, cb.to(device))
    kw = dict(user_id=uid, scale=scale)
    # the last T tokens as drafted ones, each seeing itself and those before it; then all blocks
    vis = torch.ones(T, S, dtype=torch.bool).tril(S - T)
    tree = torch.tensor([(1 << (t + 1)) - 1 for t in range(T)], dtype=torch.int64, device=device)
    tried = paged_tree_attention(*args, tree, **kw)
    blocks = torch.arange(pt.shape[1], dtype=torch.int32, device=device).expand(B, H, T, -1).contiguous()
    for got in (tried, paged_block_attention(*args, blocks, **kw)):
        assert torch.equal(got, got[:1].expand_as(got))
        most = 0.0
        for h in range(G * H):
            want, bound = P.attend(q[0, h].double(), k[0, h // G], v[0, h // G], vis, scale, dtype, False)
            P.close(got[0, h], want, bound, f"head {h}")
            s = torch.where(vis, q[0, h].double() @ k[0, h // G].T * scale, -math.inf).softmax(-1)
            most = max(most, float(s[:, [3, 17, 20]].amax()))
        assert most > 0.05                               # the weights of these tokens are no small part


def test_dual_tensors_are_refused(device):
    """A tangent would be dropped in silence: the eager and the prepared calls raise."""
    from torch.autograd import forward_ad
    from omnistack_rs.cache import (PagedBlockAttention, PagedTreeAttention, paged_block_attention, paged_tree_attention,
                                    select_blocks)
    parts, cb = P.packed(2, 2, 40, seed=411), P.codebooks(2).to(device)
    cache, pt, lt = P.paged(device, parts, 16, bounds=True)
    q = torch.randn(2, 8, 1, 128, generator=torch.Generator().manual_seed(412)).to(torch.bfloat16).to(device)
    tree = torch.ones(1, dtype=torch.int64, device=device)
    tr, bl = PagedTreeAttention(cache, cb, 8, 2, pt.shape[1]), PagedBlockAttention(cache, cb, 8, 2, pt.shape[1], 2)
    blocks = select_blocks(q, cache, pt, lt, cb, 2)
    ref = [tr.run(q, pt, lt, tree).clone(), bl.run(q, pt, lt).clone()]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: paged_tree_attention(dual, cache, pt, lt, cb, tree),
                     lambda: paged_block_attention(dual, cache, pt, lt, cb, blocks), lambda: tr.run(dual, pt, lt, tree),
                     lambda: bl.run(dual, pt, lt)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(tr.run(q, pt, lt, tree), ref[0]) and torch.equal(bl.run(q, pt, lt), ref[1])


def test_64_bit_numbers_do_not_wrap(device):
    """Lengths, page ids and draft counts of int64 beyond int32, whose low words alone would fit."""
    from omnistack_rs.cache import paged_block_attention, paged_tree_attention, select_blocks
    parts, cb = P.packed(2, 2, 40, seed=421), P.codebooks(2).to(device)
    cache, pt, lt = P.paged(device, parts, 16, bounds=True)
    q = torch.randn(2, 8, 2, 128, generator=torch.Generator().manual_seed(422)).to(torch.bfloat16).to(device)
    tree = torch.tensor([1, 3], dtype=torch.int64, device=device)
    nd = torch.tensor([2, 1], device=device)
    blocks = select_blocks(q, cache, pt, lt, cb, 2)
    ref = paged_tree_attention(q, cache, pt, lt, cb, tree, n_draft=nd)
    assert torch.equal(paged_tree_attention(q, cache, pt.long(), lt.long(), cb, tree, n_draft=nd.int()), ref)
    for far in (1 << 32, -(1 << 32), 1 << 62):
        for i in range(3):
            a = [pt.long(), lt.long(), nd.clone()]
            a[i].view(-1)[0] += far
            kw = dict(n_draft=a[2])
            with pytest.raises((ValueError, IndexError)):
                paged_tree_attention(q, cache, a[0], a[1], cb, tree, **kw)
            got = paged_tree_attention(q, cache, a[0], a[1], cb, tree, validate=False, **kw)
            assert torch.isnan(got[0]).all() and torch.equal(got[1], ref[1])
            if i < 2:
                with pytest.raises((ValueError, IndexError)):
                    select_blocks(q, cache, a[0], a[1], cb, 2)
                with pytest.raises((ValueError, IndexError)):
                    paged_block_attention(q, cache, a[0], a[1], cb, blocks)
                got = paged_block_attention(q, cache, a[0], a[1], cb, blocks, validate=False)
                assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()


def test_numbers_passed_over_may_repeat(device):
    """Any padding behind a query's blocks, the same number twice among it; one of its own blocks twice is refused."""
    from omnistack_rs.cache import paged_block_attention
    lens, T = [40, 70], 2
    parts, cb = P.packed(2, 2, 70, seed=431), P.codebooks(2).to(device)
    cache, pt, lt = P.paged(device, parts, 16, lens)
    q = torch.randn(2, 8, T, 128, generator=torch.Generator().manual_seed(432)).to(torch.bfloat16).to(device)
    blocks = torch.tensor([0, 2, -1, -1], dtype=torch.int32, device=device).expand(2, 2, T, 4).contiguous()
    ref = paged_block_attention(q, cache, pt, lt, cb, blocks)
    for pad in (-5, 3, 4, 5, 1 << 30):
        other = blocks.clone()
        other[0, :, :, 2:] = pad if pad != 5 else 3                    # sequence 0 has blocks 0 to 2
        other[1, :, :, 2:] = pad if pad > 4 else -3                    # sequence 1 has blocks 0 to 4
        assert torch.equal(paged_block_attention(q, cache, pt, lt, cb, other), ref), pad
    # block 1 of sequence 0 is the last that query 0 of 17 tokens does not see
    short = torch.tensor([17, 70], dtype=torch.int32, device=device)
    twice = torch.tensor([0, 1, 1, -1], dtype=torch.int32, device=device).expand(2, 2, T, 4).contiguous()
    twice[1], twice[0, :, 1, 2] = blocks[1], -1
    once = torch.where(twice == 1, -1, twice)
    once[0, :, 1, 1] = 1
    got = paged_block_attention(q, cache, pt, short, cb, twice)
    assert torch.equal(got, paged_block_attention(q, cache, pt, short, cb, once))
    for b, t, n in ((0, 0, 0), (0, 1, 2), (1, 0, 4), (1, 1, 4)):
        bad = blocks.clone()
        bad[b, 1, t] = torch.tensor([n, -1, n, 9], dtype=torch.int32)
        with pytest.raises(ValueError):
            paged_block_attention(q, cache, pt, lt, cb, bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,T", [(1, 1), (4, 8), (4, 12), (4, 16)])
def test_values_that_cancel(device, G, T, dtype):
    """Equal weights over values whose fp16 roundings are all that is left of them: the second term of V's centroids."""
    from omnistack_rs.cache import paged_block_attention, paged_tree_attention
    S, rest = 80, 0.49 * 2.0 ** -9                                     # less than half a step of fp16 at 2.5
    cb = torch.linspace(-2.0, 2.0, 16)
    cb[0], cb[15] = -2.5 + rest, 2.5 + rest
    vc = _same(S, 0)
    vc[1::2] = 15
    cache, pt, lt = _pool(device, _same(S, 3), vc, 16)
    q = torch.zeros(1, G, T, 128, dtype=dtype, device=device)
    none = torch.zeros(T, dtype=torch.int64, device=device)
    more = torch.cat((pt, pt[:, :4]), 1).contiguous()                  # drafted tokens that nobody sees
    trees = paged_tree_attention(q, cache, more, lt + T, cb.to(device), none, with_qjl=False)
    blocks = torch.arange(pt.shape[1], dtype=torch.int32, device=device).expand(1, 1, 1, -1).contiguous()
    picked = paged_block_attention(q[:, :, :1], cache, pt, lt, cb.to(device), blocks, with_qjl=False)
    want = (float(cb[0]) + float(cb[15])) / 2
    # the output's half step; 22 bits of a centroid in [2, 4); fp32 sums of 80 such terms
    off = torch.finfo(dtype).eps / 2 * want + 2.0 ** -20 + 80 * 2.0 ** -24 * 2.5
    assert off < want / 16
    for got in (trees, picked):
        assert float((got.double() - want).abs().max()) <= off


def test_roundings_common_to_a_codebook(device):
    """Centroids that fp16 rounds by the same share of themselves, one key against as much weight in others far below it:
    bf16 calls take the share back from the scores."""
    from omnistack_rs.cache import paged_tree_attention
    e = 0.45 * 2.0 ** -10                                              # below half a step of fp16 at a power of two
    half = 2.0 ** torch.arange(-6, 2).double() * (1 + e)
    cb = torch.cat((-half.flip(0), half)).float()
    q = torch.full((1, 1, 1, 128), 0.49, dtype=torch.bfloat16)
    gap = float(q[0, 0, 0, 0]) * 128 * (float(cb[15]) - float(cb[8])) / math.sqrt(128)
    n = round(math.exp(gap))
    assert 3e4 < n < 1e5
    kc, vc = _same(n + 1, 8), _same(n + 1, 0)
    kc[0], vc[0] = 15, 15
    cache, pt, lt = _pool(device, kc, vc, 256)
    got = paged_tree_attention(q.to(device), cache, pt, lt, cb.to(device), torch.ones(1, dtype=torch.int64, device=device),
                               with_qjl=False, validate=False).double().cpu()
    w = n * math.exp(-gap)
    want = float(cb[15]) * (1 - w) / (1 + w)
    # a share x of the others' weight moves the result by x / 2 of a value: of P's rounding 2^-12, of the scores' fp32 sums
    # 2^-16 of 11; the output's half step and V's 22 bits.  The centroids' rounding would be 11 e = 4.8e-3.
    off = float(cb[15]) * (2.0 ** -12 + 11 * 2.0 ** -16) / 2 + 2.0 ** -8 * abs(want) + 2.0 ** -20
    assert off < float(cb[15]) * gap * e / 8
    assert float((got - want).abs().max()) <= off
