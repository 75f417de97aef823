"""Attention over the blocks (pages) of the cache that a cheap score selects
for each query (omni_block_select, omni_attn_blocks).

No counterpart in the reference.  A pool made with ``bounds=True`` keeps, for
every page and kv head, the least and largest key code of each dim (one byte a
dim; a page of 16 tokens holds 140 bytes a token): with codebooks that ascend,
the largest score that any of its keys could have follows from them.
``select_blocks`` adds that bound up over a kv head's query heads, in whole
numbers, and takes the ``top`` blocks of each query token and kv head;
``paged_block_attention`` attends to those alone.  ``PagedBlockAttention`` is
both, prepared for a serving loop.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ..kernels.quantize import _prep_codebooks
from .paged import PagedKVCache
from .tree import _Prepared, aligned, check_pool, check_q, check_scale, check_tables


def _check_bounds(cache: PagedKVCache) -> None:
    b = cache.k_bounds
    if b is None:
        raise ValueError("the cache keeps no bounds: make it with PagedKVCache(..., bounds=True)")
    if b.dtype != torch.uint8 or tuple(b.shape) != (cache.n_pages, cache.n_kv_heads, cache.head_dim) or \
            not b.is_contiguous() or b.data_ptr() % 16:
        raise ValueError("cache.k_bounds must be a contiguous uint8 tensor of the pool's shape")


def _check_top(top: int, first: int, recent: int) -> None:
    if first < 0 or recent < 1 or first + recent > top:
        raise ValueError(f"need first >= 0, recent >= 1 and first + recent <= top, got {first}, {recent} and {top}")


def _ascend(cb: torch.Tensor) -> None:
    if not bool((cb[..., 1:] >= cb[..., :-1]).all()):
        raise ValueError("the bounds need codebooks that ascend")


def select_blocks(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                  codebooks: torch.Tensor, top: int, *, first: int = 1, recent: int = 1, rotate_q: bool = False,
                  sign_flip: Optional[torch.Tensor] = None, validate: bool = True) -> torch.Tensor:
    """Block numbers (positions in the page table) for each query and kv head:
    int32 (B, n_kv_heads, T, top), ascending, -1 behind the last.

    Query token t of sequence b sees the first ``seq_lens[b] - T + t + 1``
    tokens.  Of their blocks the first ``first`` and the last ``recent`` are
    taken, then those of the largest scores; the lower block wins a tie.  The
    score is the upper bound of sum_h q_h . c[code] over the kv head's query
    heads (scores are of one sign: a negative scale wants -q here) with the sums
    of q and the codebooks rounded to int8 by powers of two, so it can lie below
    the bound by what that rounds away; residual signs take no part.  Arguments
    as for ``paged_tree_attention``; ``validate`` also checks that the codebooks
    ascend."""
    check_q(q, cache)
    _check_bounds(cache)
    _check_top(top, first, recent)
    B, Hq, T, D = q.shape
    dev = _lib.require_device(q, cache.k_bounds, page_table, seq_lens)
    pt, lens = check_tables(cache, page_table, seq_lens, B, dev, validate)
    cb, per_head = _prep_codebooks(codebooks, cache.n_kv_heads, dev)
    if validate:
        _ascend(cb)
    qc = aligned(q)
    sf = aligned(_lib.sign_flip_i8(sign_flip, D, dev), 8) if (rotate_q and sign_flip is not None) else None
    blocks = torch.empty(B, cache.n_kv_heads, T, top, dtype=torch.int32, device=dev)
    L = _lib.lib()
    ws_bytes = _lib.on_device(dev, L.omni_block_select_workspace_size, B, cache.n_kv_heads, T, pt.shape[1], top)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _lib.check(_lib.on_device(
        dev, L.omni_block_select, _lib.ptr(qc), _lib.dtype_code(q.dtype), _lib.ptr(cache.k_bounds), cache.n_pages,
        cache.page_size, _lib.ptr(pt), pt.shape[1], _lib.ptr(lens), _lib.ptr(cb), per_head, B, Hq, cache.n_kv_heads, T, D, top,
        first, recent, int(rotate_q), _lib.ptr(sf), _lib.ptr(blocks), _lib.ptr(ws), ws_bytes, _lib.stream_of(dev)))
    return blocks


def paged_block_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                          codebooks: torch.Tensor, blocks: torch.Tensor, user_id: int = 0, scale: Optional[float] = None,
                          with_qjl: bool = True, *, rotate_q: bool = False, sign_flip: Optional[torch.Tensor] = None,
                          validate: bool = True) -> torch.Tensor:
    """Attention of q (B, n_heads, T, 128), float16 or bfloat16, over selected
    blocks: query token t of sequence b sees those of its first ``seq_lens[b] -
    T + t + 1`` tokens that lie in ``blocks[b, kv head, t]`` (int32, as
    ``select_blocks`` gives them, in any order; numbers outside the query's
    blocks are passed over).  Returns q's shape and dtype; a query that sees
    nothing is NaN.  ``validate`` also refuses one of its blocks named twice for
    a query, which would count twice.  No gradient."""
    _lib.refuse_tangents("paged_block_attention", q)
    check_q(q, cache)
    B, Hq, T, D = q.shape
    H = cache.n_kv_heads
    dev = _lib.require_device(q, cache.k_nibbles, page_table, seq_lens, blocks)
    check_pool(cache, with_qjl)
    pt, lens = check_tables(cache, page_table, seq_lens, B, dev, validate)
    if blocks.dim() != 4 or tuple(blocks.shape[:3]) != (B, H, T) or blocks.shape[3] < 1 or blocks.dtype != torch.int32:
        raise ValueError(f"blocks must be int32 ({B}, {H}, {T}, top), got {blocks.dtype} {tuple(blocks.shape)}")
    bl = blocks.contiguous()
    if validate and B:
        s = bl.cpu().sort(-1)[0]
        seen = (lens.cpu().to(torch.int64)[:, None] - T + 1 + torch.arange(T)).clamp_min(0)
        n = ((seen + cache.page_size - 1) // cache.page_size)[:, None, :, None]          # blocks of each query
        if bool(((s[..., 1:] == s[..., :-1]) & (s[..., 1:] >= 0) & (s[..., 1:] < n)).any()):
            raise ValueError("blocks names a block twice for one query")
    scale = check_scale(scale, D)
    cb, per_head = _prep_codebooks(codebooks, H, dev)
    qc = aligned(q)
    gb = _lib.g_bits(_lib.head_seeds(user_id, H), D, dev) if with_qjl else None
    sf = aligned(_lib.sign_flip_i8(sign_flip, D, dev), 8) if (rotate_q and sign_flip is not None) else None
    out = _lib.empty_as(q)
    L = _lib.lib()
    code, ps, top = _lib.dtype_code(q.dtype), cache.page_size, bl.shape[3]
    ws_bytes = _lib.on_device(dev, L.omni_attn_blocks_workspace_size, B, Hq, H, T, top, ps, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _lib.check(_lib.on_device(
        dev, L.omni_attn_blocks, _lib.ptr(qc), code, _lib.ptr(cache.k_nibbles), _lib.ptr(cache.k_qjl if with_qjl else None),
        _lib.ptr(cache.k_norms if with_qjl else None), _lib.ptr(cache.v_nibbles), cache.n_pages, ps, _lib.ptr(pt), pt.shape[1],
        _lib.ptr(lens), _lib.ptr(bl), top, _lib.ptr(cb), per_head, _lib.ptr(gb), B, Hq, H, T, D, scale, int(with_qjl),
        int(rotate_q), _lib.ptr(sf), _lib.ptr(out), _lib.ptr(ws), ws_bytes, _lib.stream_of(dev)))
    return out


class PagedBlockAttention(_Prepared):
    """Prepared ``select_blocks`` and ``paged_block_attention`` over one page pool
    (serving loops): ``run(q, page_table, seq_lens)`` selects each query's ``top``
    blocks, attends to them and returns the reused output, q's dtype; the
    selection is left in ``blocks``.  The pool's bounds must be those of its
    tokens (``PagedKVCache.append``, ``write`` and ``keep`` see to it).  Otherwise
    as ``PagedTreeAttention``."""

    def __init__(self, cache: PagedKVCache, codebooks: torch.Tensor, n_heads: int, batch: int, max_pages: int, top: int,
                 q_tokens: int = 1, first: int = 1, recent: int = 1, user_id: int = 0, scale: Optional[float] = None,
                 with_qjl: bool = True, q_dtype: torch.dtype = torch.bfloat16, rotate_q: bool = False,
                 sign_flip: Optional[torch.Tensor] = None):
        _check_bounds(cache)
        _check_top(top, first, recent)
        super().__init__(cache, codebooks, n_heads, batch, max_pages, q_tokens, user_id, scale, with_qjl, q_dtype, rotate_q,
                         sign_flip)
        if self.scale <= 0.0:
            raise ValueError(f"the selection needs a positive scale, got {self.scale}")
        _ascend(self.cb)
        self.blocks = torch.empty(self.B, cache.n_kv_heads, self.T, top, dtype=torch.int32, device=self.device)
        L = _lib.lib()
        select = _lib.on_device(self.device, L.omni_block_select_workspace_size, self.B, cache.n_kv_heads, self.T,
                                self.max_pages, top)
        attend = _lib.on_device(self.device, L.omni_attn_blocks_workspace_size, self.B, self.Hq, cache.n_kv_heads, self.T, top,
                                cache.page_size, _lib.dtype_code(q_dtype))
        self._make_plan(max(select, attend), cache.k_bounds, self.blocks, top, first, recent)
        self._run_fn = L.omni_attn_blocks_plan_run

    def run(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor) -> torch.Tensor:
        self._check_run(q, page_table, seq_lens)
        rc = _lib.on_device(self.device, self._run_fn, self._plan, q.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
                            _lib.stream_of(self.device))
        if rc:
            _lib.check(rc)
        return self.out
