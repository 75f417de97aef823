"""Attention of a tree of drafted tokens over the paged cache (omni_attn_tree).

No counterpart in the reference.  A server that drafts several tokens for a
sequence appends them all to its cache (``PagedKVCache.append``), asks for
every drafted token's attention in one call, and keeps those that its model
accepts (``PagedKVCache.keep``).  Drafted token t sees the cached tokens and
the drafted tokens on its path, as one of a chain would that had only those
before it; q comes rotated to the token's position in that chain
(``kernels.rope.qk_norm_rope``), with any adapter's update in it.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from .. import _lib
from ..kernels.quantize import _check_packed, _prep_codebooks
from .paged import PagedKVCache

MAX_DRAFT = 64
_DTYPES = (torch.float16, torch.bfloat16)


def tree_masks(parents: torch.Tensor) -> torch.Tensor:
    """The ``tree`` of ``paged_tree_attention`` from parents: integers (T,) or
    (B, T), ``parents[t]`` < t the drafted token that t follows, negative where
    it follows the last cached token.  int64 of the same shape; bit j of entry t
    is set for t itself and every token on its way up.  Made on the host (a copy
    and a wait where parents are on the device, not for graph capture): keep the
    masks of a tree that is used again."""
    if parents.dim() not in (1, 2) or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"parents must be int32 or int64 (T,) or (B, T), got {parents.dtype} {tuple(parents.shape)}")
    T = parents.shape[-1]
    if not 1 <= T <= MAX_DRAFT:
        raise ValueError(f"1 to {MAX_DRAFT} drafted tokens, got {T}")
    host = parents.cpu().to(torch.int64)
    if bool((host >= torch.arange(T)).any()):
        raise ValueError("a parent must come before its child")
    rows = []
    for row in host.reshape(-1, T).tolist():
        m = []
        for t, p in enumerate(row):
            m.append((1 << t) | (m[p] if p >= 0 else 0))
        rows.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(rows, dtype=torch.int64).reshape(parents.shape).to(parents.device)


def aligned(t: Optional[torch.Tensor], to: int = 16) -> Optional[torch.Tensor]:
    """`t`, or a contiguous copy where it is not contiguous or not at a multiple of `to` bytes."""
    if t is None or (t.is_contiguous() and t.data_ptr() % to == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def check_pool(cache: PagedKVCache, with_qjl: bool) -> torch.device:
    """The pool's arrays as the kernels read them."""
    _check_packed(cache.k_nibbles, cache.k_qjl if with_qjl else None, cache.k_norms if with_qjl else None, "cache.k_nibbles")
    if cache.v_nibbles.dtype != torch.uint8 or cache.v_nibbles.shape != cache.k_nibbles.shape:
        raise ValueError("cache.v_nibbles must be uint8 of cache.k_nibbles' shape")
    if with_qjl and cache.k_norms.dtype != torch.float32:
        raise ValueError(f"cache.k_norms must be float32, got {cache.k_norms.dtype}")
    if tuple(cache.k_nibbles.shape) != (cache.n_pages, cache.n_kv_heads, cache.page_size, cache.head_dim // 2):
        raise ValueError(f"cache.k_nibbles does not have the pool's shape: {tuple(cache.k_nibbles.shape)}")
    used = (cache.k_nibbles, cache.v_nibbles) + ((cache.k_qjl, cache.k_norms) if with_qjl else ())
    if any(not t.is_contiguous() or t.data_ptr() % 16 for t in used):
        raise ValueError("the cache's arrays must be contiguous and start at multiples of 16 bytes")
    return _lib.require_device(*used)


def check_scale(scale: Optional[float], head_dim: int) -> float:
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not abs(scale) <= 2.3e38:                     # the kernels multiply it by log2 e
        raise ValueError(f"scale must be finite and at most 2.3e38 in size, got {scale}")
    return scale


def check_q(q: torch.Tensor, cache: PagedKVCache) -> None:
    if q.dim() != 4 or q.shape[3] != cache.head_dim:
        raise ValueError(f"q must be (B, n_heads, T, {cache.head_dim}), got {tuple(q.shape)}")
    if q.dtype not in _DTYPES:
        raise ValueError(f"q must be float16 or bfloat16 (float32: paged_attention), got {q.dtype}")
    if q.shape[1] < 1 or q.shape[1] % cache.n_kv_heads:
        raise ValueError(f"n_heads={q.shape[1]} must be a multiple of n_kv_heads={cache.n_kv_heads}")
    if not 1 <= q.shape[2] <= MAX_DRAFT:
        raise ValueError(f"1 to {MAX_DRAFT} query tokens, got {q.shape[2]}")


def as_int32(t: torch.Tensor) -> torch.Tensor:
    """Contiguous int32; what int32 does not hold stays out of every range (lengths, page ids and counts are not negative)."""
    return (t.clamp(-1, 2 ** 31 - 1) if t.dtype == torch.int64 else t).to(dtype=torch.int32).contiguous()


def check_tables(cache, page_table, seq_lens, B, dev, validate):
    """Page table and lengths as contiguous int32, checked on the host where asked."""
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.shape[1] < 1:
        raise ValueError(f"page_table must be ({B}, max_pages), got {tuple(page_table.shape)}")
    pt, lens = as_int32(page_table), as_int32(seq_lens.reshape(-1))
    if lens.numel() != B:
        raise ValueError(f"seq_lens must have {B} entries, got {lens.numel()}")
    if validate and B:
        lh, th, ps = lens.cpu().to(torch.int64), pt.cpu(), cache.page_size
        if int(lh.min()) < 0 or int(lh.max()) > pt.shape[1] * ps:
            raise ValueError(f"seq_lens must lie in [0, {pt.shape[1] * ps}] (the page table's width)")
        used = torch.arange(pt.shape[1])[None, :] < ((lh + ps - 1) // ps)[:, None]
        bad = used & ((th < 0) | (th >= cache.n_pages))
        if bool(bad.any()):
            raise IndexError(f"sequence {int(bad.nonzero()[0][0])}: page id out of range for a pool of {cache.n_pages} pages")
    return pt, lens


def paged_tree_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                         codebooks: torch.Tensor, tree: torch.Tensor, user_id: int = 0, scale: Optional[float] = None,
                         with_qjl: bool = True, *, n_draft: Optional[torch.Tensor] = None, rotate_q: bool = False,
                         sign_flip: Optional[torch.Tensor] = None, validate: bool = True) -> torch.Tensor:
    """Attention of T <= 64 drafted tokens per sequence, q (B, n_heads, T, 128)
    in float16 or bfloat16; returns that shape in q's dtype.

    ``seq_lens`` counts the drafted tokens, which are the sequence's last
    ``n_draft[b]`` (default T).  Drafted token t sees every token before them,
    and drafted token j where bit j of ``tree[b, t]`` (int64 (B, T), or (T,) for
    all sequences; ``tree_masks`` makes it from parents) is set, itself included
    only if its own bit is.  Rows t >= n_draft[b] are zeros; a row that sees
    nothing is NaN.  ``rotate_q`` applies the signed Hadamard rotation of the
    cache to q, not rounded to q's dtype in between.  Scores are fp32 and meant
    for sizes far below 2^24; past it outputs may not be finite.  With ``validate`` lengths,
    page ids and draft counts that do not fit raise (device-to-host copies);
    without it the rows of such sequences are NaN.  No gradient."""
    _lib.refuse_tangents("paged_tree_attention", q)
    check_q(q, cache)
    B, Hq, T, D = q.shape
    dev = _lib.require_device(q, cache.k_nibbles, page_table, seq_lens, tree, n_draft)
    check_pool(cache, with_qjl)
    pt, lens = check_tables(cache, page_table, seq_lens, B, dev, validate)
    if tree.dtype != torch.int64 or tuple(tree.shape) not in ((T,), (B, T)):
        raise ValueError(f"tree must be int64 ({T},) or ({B}, {T}), got {tree.dtype} {tuple(tree.shape)}")
    tr = tree.contiguous()
    nd = None
    if n_draft is not None:
        if n_draft.numel() != B:
            raise ValueError(f"n_draft must have {B} entries, got {n_draft.numel()}")
        nd = as_int32(n_draft.reshape(-1))
    if validate and B:
        n = torch.full((B,), T) if nd is None else nd.cpu().to(torch.int64)
        if bool(((n < 0) | (n > T) | (n > lens.cpu())).any()):
            raise ValueError(f"n_draft must lie in [0, {T}] and not exceed seq_lens")
    scale = check_scale(scale, D)
    cb, per_head = _prep_codebooks(codebooks, cache.n_kv_heads, dev)
    qc = aligned(q)
    gb = _lib.g_bits(_lib.head_seeds(user_id, cache.n_kv_heads), D, dev) if with_qjl else None
    sf = aligned(_lib.sign_flip_i8(sign_flip, D, dev), 8) if (rotate_q and sign_flip is not None) else None
    out = _lib.empty_as(q)
    L = _lib.lib()
    code, ps, mp = _lib.dtype_code(q.dtype), cache.page_size, pt.shape[1]
    ws_bytes = _lib.on_device(dev, L.omni_attn_tree_workspace_size, B, Hq, cache.n_kv_heads, T, mp, ps, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _lib.check(_lib.on_device(
        dev, L.omni_attn_tree, _lib.ptr(qc), code, _lib.ptr(cache.k_nibbles), _lib.ptr(cache.k_qjl if with_qjl else None),
        _lib.ptr(cache.k_norms if with_qjl else None), _lib.ptr(cache.v_nibbles), cache.n_pages, ps, _lib.ptr(pt), mp,
        _lib.ptr(lens), _lib.ptr(nd), _lib.ptr(tr), T if tr.dim() == 2 else 0, _lib.ptr(cb), per_head, _lib.ptr(gb), B, Hq,
        cache.n_kv_heads, T, D, scale, int(with_qjl), int(rotate_q), _lib.ptr(sf), _lib.ptr(out), _lib.ptr(ws), ws_bytes,
        _lib.stream_of(dev)))
    return out


class _Prepared:
    """What the prepared forms share: the pool, codebooks, G, output and
    workspace held once, and a native plan that names them."""

    def __init__(self, cache, codebooks, n_heads, batch, max_pages, q_tokens, user_id, scale, with_qjl, q_dtype, rotate_q,
                 sign_flip):
        H, D = cache.n_kv_heads, cache.head_dim
        if n_heads < 1 or n_heads % H:
            raise ValueError(f"n_heads={n_heads} must be a multiple of n_kv_heads={H}")
        if q_dtype not in _DTYPES:
            raise ValueError(f"q_dtype must be float16 or bfloat16, got {q_dtype}")
        self.cache, self.B, self.Hq, self.T, self.max_pages = cache, int(batch), int(n_heads), int(q_tokens), int(max_pages)
        if self.B < 0 or not 1 <= self.T <= MAX_DRAFT or self.max_pages < 1:
            raise ValueError(f"batch must be >= 0, q_tokens 1 to {MAX_DRAFT} and max_pages >= 1")
        self.device = check_pool(cache, with_qjl)
        self.scale = check_scale(scale, D)
        self.cb, self.per_head = _prep_codebooks(codebooks, H, self.device)
        self.gb = _lib.g_bits(_lib.head_seeds(user_id, H), D, self.device) if with_qjl else None
        self.sf = aligned(_lib.sign_flip_i8(sign_flip, D, self.device), 8) if (rotate_q and sign_flip is not None) else None
        self.q_dtype, self.with_qjl, self.rotate_q = q_dtype, bool(with_qjl), bool(rotate_q)
        self._shape = (self.B, self.Hq, self.T, D)
        self._pt_shape = (self.B, self.max_pages)
        self.out = torch.empty(self._shape, dtype=q_dtype, device=self.device)

    def _make_plan(self, ws_bytes, bounds=None, blocks=None, top=0, first=0, recent=0):
        c = self.cache
        self.ws_bytes = ws_bytes
        self.ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=self.device)
        # the plan's addresses stay valid while these are held
        self._held = (c.k_nibbles, c.k_qjl, c.k_norms, c.v_nibbles, bounds, blocks)
        self._plan = ctypes.c_void_p()
        L = _lib.lib()
        _lib.check(L.omni_attn_pages_plan_create(
            _lib.dtype_code(self.q_dtype), _lib.ptr(c.k_nibbles), _lib.ptr(c.k_qjl if self.with_qjl else None),
            _lib.ptr(c.k_norms if self.with_qjl else None), _lib.ptr(c.v_nibbles), _lib.ptr(bounds), c.n_pages, c.page_size,
            self.max_pages, _lib.ptr(blocks), top, first, recent, _lib.ptr(self.cb), self.per_head, _lib.ptr(self.gb), self.B,
            self.Hq, c.n_kv_heads, self.T, self.scale, int(self.with_qjl), int(self.rotate_q), _lib.ptr(self.sf),
            _lib.ptr(self.out), _lib.ptr(self.ws), ws_bytes, ctypes.byref(self._plan)))
        self._destroy = L.omni_attn_pages_plan_destroy

    def _check_run(self, q, page_table, seq_lens):
        """Host-only checks (no device work, safe under graph capture)."""
        _lib.refuse_tangents(type(self).__name__, q)
        if q.shape != self._shape or q.dtype != self.q_dtype or not q.is_contiguous() or q.data_ptr() % 16:
            raise ValueError(f"q must be a contiguous {self.q_dtype} tensor of shape {self._shape} at a multiple of 16 bytes")
        if page_table.shape != self._pt_shape or page_table.dtype != torch.int32 or not page_table.is_contiguous():
            raise ValueError(f"page_table must be a contiguous int32 tensor of shape {self._pt_shape}")
        if seq_lens.dtype != torch.int32 or seq_lens.numel() != self.B or not seq_lens.is_contiguous():
            raise ValueError(f"seq_lens must be a contiguous int32 tensor of {self.B} entries")
        if q.device != self.device or page_table.device != self.device or seq_lens.device != self.device:
            raise ValueError(f"q, page_table and seq_lens must be on {self.device}")

    def __del__(self):
        plan = getattr(self, "_plan", None)
        if plan is not None and plan.value:
            self._destroy(plan)
            self._plan = None


class PagedTreeAttention(_Prepared):
    """Prepared ``paged_tree_attention`` over one page pool (serving loops).

    Converts codebooks, uploads G and allocates the output and workspace once
    for ``batch`` sequences of ``q_tokens`` drafted tokens and page tables
    ``max_pages`` wide; ``run(q, page_table, seq_lens, tree, n_draft)`` then
    enqueues the kernels on the current stream (no host sync, no allocation:
    safe to capture in a HIP graph) and returns the reused output, q's dtype.
    Runs of one object that may overlap (two streams, two captured graphs) share
    that output and workspace: give each an object of its own.  Tensors are
    taken as they are (contiguous, on the pool's device, int32 tables, lengths
    and counts, int64 trees) and nothing of their values is checked on the host:
    sequences whose page ids or lengths do not fit give NaN rows."""

    def __init__(self, cache: PagedKVCache, codebooks: torch.Tensor, n_heads: int, batch: int, max_pages: int,
                 q_tokens: int = 1, user_id: int = 0, scale: Optional[float] = None, with_qjl: bool = True,
                 q_dtype: torch.dtype = torch.bfloat16, rotate_q: bool = False, sign_flip: Optional[torch.Tensor] = None):
        super().__init__(cache, codebooks, n_heads, batch, max_pages, q_tokens, user_id, scale, with_qjl, q_dtype, rotate_q,
                         sign_flip)
        L = _lib.lib()
        self._make_plan(_lib.on_device(self.device, L.omni_attn_tree_workspace_size, self.B, self.Hq, cache.n_kv_heads, self.T,
                                       self.max_pages, cache.page_size, _lib.dtype_code(q_dtype)))
        self._run_fn = L.omni_attn_tree_plan_run

    def run(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, tree: torch.Tensor,
            n_draft: Optional[torch.Tensor] = None) -> torch.Tensor:
        self._check_run(q, page_table, seq_lens)
        one = tree.dim() == 1
        if tree.dtype != torch.int64 or tree.shape != ((self.T,) if one else (self.B, self.T)) or not tree.is_contiguous() or \
                tree.device != self.device:
            raise ValueError(f"tree must be a contiguous int64 tensor of shape ({self.T},) or ({self.B}, {self.T}) on "
                             f"{self.device}")
        if n_draft is not None and (n_draft.dtype != torch.int32 or n_draft.numel() != self.B or not n_draft.is_contiguous() or
                                    n_draft.device != self.device):
            raise ValueError(f"n_draft must be a contiguous int32 tensor of {self.B} entries on {self.device}")
        rc = _lib.on_device(self.device, self._run_fn, self._plan, q.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(),
                            tree.data_ptr(), 0 if one else self.T, _lib.ptr(n_draft), _lib.stream_of(self.device))
        if rc:
            _lib.check(rc)
        return self.out
