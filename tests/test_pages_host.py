"""The attention over drafted tokens' trees and selected blocks: what is decided
on the host (CPU only: masks, argument checks, workspace sizes)."""
import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from omnistack_rs import _lib
    return _lib.lib()


def test_tree_masks():
    from omnistack_rs.cache import tree_masks
    m = tree_masks(torch.tensor([-1, 0, 0, 1, -1, 4]))
    assert m.tolist() == [1, 3, 5, 11, 16, 48] and m.dtype == torch.int64
    chain = tree_masks(torch.arange(-1, 63, dtype=torch.int32).expand(2, 64))
    assert chain.shape == (2, 64) and chain[1].tolist() == [(1 << (t + 1)) - 1 for t in range(63)] + [-1]
    assert tree_masks(torch.full((1, 1), -5)).tolist() == [[1]]
    star = tree_masks(torch.full((64,), -1))
    assert star[63] == -(1 << 63)
    for bad in (torch.tensor([0]), torch.tensor([-1, 1]), torch.tensor([-1, 2, 0]), torch.arange(-1, 64), torch.zeros(0).long(),
                torch.tensor([-1.0]), torch.tensor(-1), torch.full((1, 1, 1), -1)):
        with pytest.raises(ValueError):
            tree_masks(bad)


def _tree(L, q=1, dt=2, nib=1, qjl=1, n_pages=8, ps=16, pt=1, mp=4, lens=1, tree=1, stride=0, gb=1, B=1, Hq=4, Hkv=2, T=3, D=128,
          scale=1.0, out=1, ws=None, wsb=0):
    return L.omni_attn_tree(q, dt, nib, qjl, nib, nib, n_pages, ps, pt, mp, lens, None, tree, stride, nib, 0, gb, B, Hq, Hkv, T,
                            D, scale, 1, 0, None, out, ws, wsb, None)


def _blocks(L, blocks=1, top=2, B=1, Hq=4, Hkv=2, T=1, mp=4, ps=16, scale=1.0, ws=None, wsb=0):
    return L.omni_attn_blocks(1, 2, 1, 1, 1, 1, 8, ps, 1, mp, 1, blocks, top, 1, 0, 1, B, Hq, Hkv, T, 128, scale, 1, 0, None, 1,
                              ws, wsb, None)


def _select(L, q=1, dt=2, B=1, Hq=4, Hkv=2, T=1, D=128, ps=16, mp=40, n_pages=8, top=4, first=1, recent=1, blocks=1, ws=None,
            wsb=0):
    return L.omni_block_select(q, dt, 1, n_pages, ps, 1, mp, 1, 1, 0, B, Hq, Hkv, T, D, top, first, recent, 0, None, blocks, ws,
                               wsb, None)


def test_entries_refuse_before_any_device_work(L):
    from omnistack_rs import _lib
    for kw, word in ((dict(dt=0), "float16"), (dict(D=64), "head_dim"), (dict(Hq=5), "multiple"), (dict(T=0), "query tokens"),
                     (dict(T=65), "query tokens"), (dict(Hq=4098, Hkv=2), "1024"), (dict(Hkv=4097, Hq=4097), "4096"),
                     (dict(B=1 << 19), "at most"), (dict(B=-1), "B >= 0"), (dict(scale=float("inf")), "scale"),
                     (dict(scale=float("nan")), "scale"), (dict(q=None), "NULL"), (dict(gb=None), "with_qjl"),
                     (dict(qjl=None), "with_qjl"), (dict(ps=8), "page_size"), (dict(ps=48), "page_size"), (dict(n_pages=0), "n_pages"),
                     (dict(n_pages=1 << 27), "pool"), (dict(mp=1 << 27), "max_pages"), (dict(tree=None), "tree"),
                     (dict(stride=2), "tree_stride"), (dict(pt=None), "page table"), (dict(lens=None), "lengths")):
        assert _tree(L, **kw) == _lib.OMNI_EINVAL and word in _lib.last_error(), (kw, _lib.last_error())
    for kw, word in ((dict(blocks=None), "blocks"), (dict(top=0), "top"), (dict(top=1 << 27), "top"), (dict(T=65), "query tokens"),
                     (dict(ps=8), "page_size")):
        assert _blocks(L, **kw) == _lib.OMNI_EINVAL and word in _lib.last_error(), (kw, _lib.last_error())
    for kw, word in ((dict(dt=0), "float16"), (dict(D=64), "head_dim"), (dict(Hq=3), "multiple"), (dict(T=65), "query tokens"),
                     (dict(B=65536), "65535"), (dict(Hq=2050), "1024"), (dict(first=-1), "first"), (dict(recent=0), "recent"),
                     (dict(first=4), "first + recent"), (dict(top=1 << 27, first=0), "top"), (dict(blocks=None), "NULL"),
                     (dict(q=None), "NULL"), (dict(ps=17), "page_size")):
        assert _select(L, **kw) == _lib.OMNI_EINVAL and word in _lib.last_error(), (kw, _lib.last_error())
    pool = (8, 2, 16)
    assert L.omni_block_bounds(1, None, *pool, 1, 4, 1, None, 3, 1, None) == _lib.OMNI_EINVAL
    assert L.omni_block_bounds(1, 1, *pool, 1, 4, 1, None, 3, 65536, None) == _lib.OMNI_EINVAL
    assert L.omni_block_bounds(1, 1, *pool, 1, 4, 1, None, -3, 1, None) == _lib.OMNI_EINVAL
    assert L.omni_cache_keep(1, 1, 1, 1, None, *pool, 1, 4, 1, 1, 1, 65, None) == _lib.OMNI_EINVAL
    assert L.omni_cache_keep(1, 1, 1, 1, None, *pool, None, 4, 1, 1, 1, 3, None) == _lib.OMNI_EINVAL
    assert L.omni_attn_tree_plan_run(None, 1, 1, 1, 1, 0, None, None) == _lib.OMNI_EINVAL
    assert L.omni_attn_blocks_plan_run(None, 1, 1, 1, None) == _lib.OMNI_EINVAL


def test_nothing_to_do(L):
    assert _tree(L, B=0) == 0 and _blocks(L, B=0) == 0 and _select(L, B=0) == 0
    assert L.omni_block_bounds(1, 1, 8, 2, 16, 1, 4, 1, None, 0, 3, None) == 0
    assert L.omni_block_bounds(1, 1, 8, 2, 16, 1, 4, 1, None, 5, 0, None) == 0
    assert L.omni_cache_keep(1, 1, 1, 1, 1, 8, 2, 16, 1, 4, 1, 1, 3, 0, None) == 0
    L.omni_attn_pages_plan_destroy(None)


def test_workspaces(L):
    from omnistack_rs import _lib
    # a long list of few rows is split: a call without its workspace, or with too little, is refused
    need = L.omni_attn_tree_workspace_size(1, 4, 2, 3, 4096, 64, 2)
    assert need > 0 and need % (2 * 6 * 132 * 4) == 0            # 2 lists of 6 rows, 132 floats a split
    for ws, wsb in ((None, 0), (None, need), (1, need - 1)):
        assert _tree(L, n_pages=8192, ps=64, mp=4096, ws=ws, wsb=wsb) == _lib.OMNI_EWORKSPACE
    need = L.omni_attn_blocks_workspace_size(1, 4, 2, 1, 2048, 64, 2)
    assert need > 0 and _blocks(L, top=2048, ps=64, mp=4096, ws=1, wsb=need - 4) == _lib.OMNI_EWORKSPACE
    assert L.omni_attn_tree_workspace_size(1, 4, 2, 3, 4, 16, 2) == 0
    need = L.omni_block_select_workspace_size(1, 2, 1, 4000, 4)
    assert need == 2 * 4000 * 4 and _select(L, mp=4000, ws=1, wsb=need - 1) == _lib.OMNI_EWORKSPACE
    assert L.omni_block_select_workspace_size(1, 2, 1, 1024, 4) == 0
    assert L.omni_block_select_workspace_size(64, 8, 1, 14336, 4) == 0                  # rows fill the chip: scores in LDS
    assert L.omni_block_select_workspace_size(64, 8, 1, 14337, 4) == 64 * 8 * 14337 * 4
    for args in ((0, 4, 2, 3, 40, 16, 2), (1, 5, 2, 3, 40, 16, 2), (1, 4, 2, 65, 40, 16, 2), (1, 4, 0, 3, 40, 16, 2),
                 (1 << 40, 4, 2, 3, 40, 16, 2), (1, 1 << 30, 1, 64, 40, 16, 2), (1, 4, 2, 3, 1 << 60, 16, 2), (1, 4, 2, 3, 40, 0, 2)):
        assert L.omni_attn_tree_workspace_size(*args) == 0


def test_cpu_tensors_are_refused():
    from omnistack_rs.cache import PagedBlockAttention, PagedKVCache, PagedTreeAttention, paged_tree_attention, select_blocks
    cache = PagedKVCache(4, 2, 16, device="cpu", bounds=True)
    assert cache.k_bounds.shape == (4, 2, 128) and PagedKVCache(4, 2, 16, device="cpu").k_bounds is None
    q, pt, lens = torch.zeros(1, 4, 1, 128, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.tensor([3])
    cb = torch.linspace(-1, 1, 16)
    for call in (lambda: paged_tree_attention(q, cache, pt, lens, cb, torch.ones(1, dtype=torch.int64)),
                 lambda: select_blocks(q, cache, pt, lens, cb, 2), lambda: PagedTreeAttention(cache, cb, 4, 1, 2),
                 lambda: PagedBlockAttention(cache, cb, 4, 1, 2, 2),
                 lambda: cache.keep(pt, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)),
                 lambda: cache.update_bounds(pt, torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))):
        with pytest.raises((ValueError, RuntimeError)):
            call()
