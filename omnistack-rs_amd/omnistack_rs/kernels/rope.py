"""Norm of query and key heads with the rotation by position, on gfx950
(omni_qk_norm_rope, omni_qk_norm_rope_backward).

No counterpart in the reference, whose caches hold keys as its callers made
them: this is the step between a model's projections and ``rotate_kv_cache``
/ ``PagedKVCache.append`` (keys) or ``omni_attn`` / ``prompt_attention``
(queries).  For every token and head of q and k, in fp32 with one rounding at
the end:

    z = x * w / sqrt(mean(x^2) + eps)          (z = x without weights)
    (z_i, z_i') turned by positions[axis_i] * inv_freq_i

over the pairs of the first ``rotary_dim`` dims; dims behind them keep z.
Positions are integers of 32 or 64 bits.  An angle is an integer product, its
whole turns gone by overflow; the frequency's rounding costs |position| 2^-65
turns, 2e-7 radians at 2^40 (about what fp32 cosines err by), 2e-4 at 2^50 and
0.2 at 2^60.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from .. import _lib
from .hadamard import HEAD_DIM

_HEAD_DIMS = (32, 64, 128, 256)
# 2^64 / 2 pi, times 2^64
_TURNS = 54157620742477409023451113735280473968


class RotaryEmbedding:
    """Frequencies of a position rotation, prepared on the device once.

    ``inv_freq``: the ``rotary_dim / 2`` angles per position (default
    ``base ** (-2 i / rotary_dim)``).  ``interleaved``: pairs are neighbours
    (2i, 2i + 1) instead of the halves (i, i + rotary_dim / 2).  Several
    position axes (time, height, width) share the pairs: ``sections`` gives
    each axis its number of pairs in turn, ``pair_axes`` names each pair's
    axis; ``n_axes`` is then the number of position rows.
    """

    def __init__(self, head_dim: int = HEAD_DIM, base: float = 10000.0, *, rotary_dim: Optional[int] = None,
                 inv_freq: Optional[Sequence[float]] = None, sections: Optional[Sequence[int]] = None,
                 pair_axes: Optional[Sequence[int]] = None, interleaved: bool = False, device="cuda"):
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        R = head_dim if rotary_dim is None else int(rotary_dim)
        if R < 0 or R > head_dim or R % 8:
            raise ValueError(f"rotary_dim must be a multiple of 8 up to head_dim {head_dim}, got {R}")
        n = R // 2
        if inv_freq is None:
            if not 0.0 < float(base) < float("inf"):
                raise ValueError(f"base must be positive and finite, got {base}")
            inv_freq = [float(base) ** (-i / n) for i in range(n)]
        freq = [float(f) for f in (inv_freq.tolist() if isinstance(inv_freq, torch.Tensor) else inv_freq)]
        if len(freq) != n or any(f != f or abs(f) == float("inf") for f in freq):
            raise ValueError(f"inv_freq must hold {n} finite values")
        if sections is not None and pair_axes is not None:
            raise ValueError("give sections or pair_axes, not both")
        if sections is not None:
            if any(int(s) < 0 for s in sections) or sum(int(s) for s in sections) != n:
                raise ValueError(f"sections must be >= 0 and sum to {n} pairs, got {list(sections)}")
            axes = [a for a, s in enumerate(sections) for _ in range(int(s))]
            self.n_axes = len(sections)
        else:
            axes = [0] * n if pair_axes is None else [int(a) for a in pair_axes]
            if len(axes) != n:
                raise ValueError(f"pair_axes must name the axis of {n} pairs, got {len(axes)}")
            self.n_axes = max(axes, default=0) + 1
        if any(a < 0 or a > 255 for a in axes) or not 1 <= self.n_axes <= 256:
            raise ValueError("position axes must lie in [0, 255]")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, R, bool(interleaved)
        # fractions of a turn per position, 64 bits, as the int64 with the same
        # bits, and behind them the axes' bytes: one upload
        turns = []
        for f in freq:
            num, den = f.as_integer_ratio()
            turns.append(((2 * num * _TURNS // (den << 64) + 1 >> 1) + (1 << 63)) % (1 << 64) - (1 << 63))
        axis_bytes = bytes(axes) + bytes(-n % 8)
        words = [int.from_bytes(axis_bytes[i:i + 8], "little", signed=True) for i in range(0, n, 8)]
        both = torch.tensor(turns + words, dtype=torch.int64).to(device)
        self.turns, self.pair_axes = both[:n], both[n:].view(torch.uint8)[:n]
        self.device = both.device


def _heads(t: torch.Tensor) -> torch.Tensor:
    """`t` as the kernels read it: the last dim contiguous, 16-byte steps."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        st = t.stride()
        if st[-1] == 1:
            step = 16 // t.element_size()
            for s, n in zip(st[:-1], t.shape):
                if s % step and n > 1:
                    break
            else:
                return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """Element strides (batch, token, head) of (N, H, D) or (B, H, T, D)."""
    s = t.stride()
    if 1 in t.shape:
        s = tuple(0 if n == 1 else st for n, st in zip(t.shape, s))
    return _lib.I64x3(0, s[0], s[1]) if len(s) == 3 else _lib.I64x3(s[0], s[2], s[1])


def _check(q, k, positions, rotary, q_weight, k_weight, eps):
    """(device, (batch, tokens), positions as (axes, tokens) or (axes, batch, tokens))."""
    qs, ks = q.shape, k.shape
    packed = len(qs) == 3
    if not (packed or len(qs) == 4) or len(ks) != len(qs):
        raise ValueError(f"q and k must be (N, heads, head_dim) or (B, heads, T, head_dim), got {tuple(qs)} "
                         f"and {tuple(ks)}")
    if not isinstance(rotary, RotaryEmbedding):
        raise TypeError("rotary must be a RotaryEmbedding")
    D = rotary.head_dim
    rows, krows = ((1, qs[0]), (1, ks[0])) if packed else ((qs[0], qs[2]), (ks[0], ks[2]))
    if qs[-1] != D or ks[-1] != D or rows != krows or qs[1] < 1 or ks[1] < 1:
        raise ValueError(f"q {tuple(qs)} and k {tuple(ks)} must agree but for their heads and have head_dim {D}")
    if q.dtype != k.dtype:
        raise ValueError(f"q and k must share a dtype, got {q.dtype} and {k.dtype}")
    if rotary.rotary_dim % (8 if _lib.dtype_code(q.dtype) == 0 else 16):
        raise ValueError(f"rotary_dim must be a multiple of {8 if q.dtype == torch.float32 else 16} for {q.dtype}, "
                         f"got {rotary.rotary_dim}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight must be given together")
    if q_weight is not None:
        _lib.dtype_code(q_weight.dtype)
        for w in (q_weight, k_weight):
            if w.dim() != 1 or w.shape[0] != D or w.dtype != q_weight.dtype:
                raise ValueError(f"q_weight and k_weight must be ({D},) of one dtype, got {w.dtype} {tuple(w.shape)}")
        if not eps >= 0.0:
            raise ValueError(f"eps must be >= 0, got {eps}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    want = (rotary.n_axes, rows[1]) if packed else (rotary.n_axes, *rows)
    if positions.shape != want:
        try:
            positions = positions.expand(want)
        except RuntimeError:
            raise ValueError(f"positions must broadcast to {want}, got {tuple(positions.shape)}") from None
    dev = _lib.require_device(q, k, positions, q_weight, k_weight)
    if dev != rotary.device:
        raise ValueError(f"rotary is on {rotary.device}, q on {dev}")
    return dev, rows, positions


def _common(q, k, pos, rotary, wq, wk, eps, rows):
    """The arguments that both directions share, behind the tensors."""
    ps = pos.stride()
    return (_lib.dtype_code(q.dtype), *rows, q.shape[1], k.shape[1], rotary.head_dim, pos.data_ptr(),
            int(pos.dtype == torch.int64), _lib.I64x3(ps[0], 0 if len(ps) == 2 else ps[1], ps[-1]),
            rotary.turns.data_ptr(), rotary.pair_axes.data_ptr(), rotary.rotary_dim, int(rotary.interleaved),
            _lib.ptr(wq), _lib.ptr(wk), 0 if wq is None else _lib.dtype_code(wq.dtype), eps)


def _forward(q, k, pos, rotary, wq, wk, eps, rows, dev, out):
    qc, kc = _heads(q), _heads(k)
    if wq is not None:
        wq, wk = _heads(wq), _heads(wk)
    if out is not None:
        qo, ko = out
    else:
        qo, ko = _lib.empty_as(q), _lib.empty_as(k)
    rc = _lib.on_device(
        dev, _lib.lib().omni_qk_norm_rope, qc.data_ptr(), _strides(qc), kc.data_ptr(), _strides(kc),
        *_common(qc, kc, pos, rotary, wq, wk, eps, rows),
        qo.data_ptr(), _strides(qo), ko.data_ptr(), _strides(ko), _lib.stream_of(dev))
    if rc:
        _lib.check(rc)
    return qo, ko


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, rotary, wq, wk, eps, rows, dev):
        # without a norm the gradient needs neither q nor k
        ctx.save_for_backward(pos, *((q, k, wq, wk) if wq is not None else ()))
        ctx.rotary, ctx.eps, ctx.rows, ctx.dev = rotary, eps, rows, dev
        return _forward(q, k, pos, rotary, wq, wk, eps, rows, dev, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        _lib.refuse_tangents("qk_norm_rope's gradient", gq, gk)
        pos, *rest = ctx.saved_tensors
        q, k, wq, wk = rest if rest else (gq, gk, None, None)
        dev, norm = ctx.dev, bool(rest)
        gq, gk = _heads(gq), _heads(gk)
        q, k = _heads(q), _heads(k)
        wqc, wkc = (None if w is None else _heads(w) for w in (wq, wk))
        dq, dk = _lib.empty_as(q), _lib.empty_as(k)
        dwq, dwk = (torch.empty_like(wqc), torch.empty_like(wkc)) if norm else (None, None)
        L = _lib.lib()
        ws_bytes = L.omni_qk_norm_rope_backward_workspace_size(ctx.rotary.head_dim) if norm else 0
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        _lib.check(_lib.on_device(
            dev, L.omni_qk_norm_rope_backward, q.data_ptr(), _strides(q), k.data_ptr(), _strides(k),
            *_common(q, k, pos, ctx.rotary, wqc, wkc, ctx.eps, ctx.rows),
            gq.data_ptr(), _strides(gq), gk.data_ptr(), _strides(gk), dq.data_ptr(), _strides(dq), dk.data_ptr(),
            _strides(dk), _lib.ptr(dwq), _lib.ptr(dwk), _lib.ptr(ws), ws_bytes, _lib.stream_of(dev)))
        return dq, dk, None, None, dwq, dwk, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: RotaryEmbedding,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *,
                 out: Optional[tuple] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm (with weights) and position rotation of q and k, one launch.

    q (N, n_heads, head_dim) and k (N, n_kv_heads, head_dim), tokens packed, or
    (B, heads, T, head_dim), the layout of the cache's encoder; float32,
    float16 or bfloat16, any strides (slices of a fused projection's output are
    read in place; a last dim that is not contiguous, or rows off 16 bytes, are
    copied first). ``positions`` int32 or int64, broadcast to (n_axes, N) or
    (n_axes, B, T): one row for text, one per axis for images and video, or one
    for all axes. ``q_weight`` / ``k_weight`` (head_dim,): the norms' weights;
    without them heads are rotated only. Returns (q', k') in the inputs' dtype,
    contiguous, or ``out`` (two tensors of the inputs' shapes; the inputs
    themselves turn in place). Gradients for q, k and the weights, once and in
    reverse mode (dual tensors are refused), all of them whichever are asked
    for; ``out`` is for calls that need none. Forward and backward can be
    captured in a HIP graph once no eager autograd graph of the same leaves is
    alive: one through these operators on the default stream is refused, as is
    one of leaves passed to them directly."""
    eps = float(eps)
    _lib.refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, *(() if out is None else out))
    dev, rows, pos = _check(q, k, positions, rotary, q_weight, k_weight, eps)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (
        q_weight is not None and (q_weight.requires_grad or k_weight.requires_grad)))
    if out is not None:
        if grad or torch.is_grad_enabled() and any(t.requires_grad for t in out):
            raise ValueError("out= takes no gradient: call it under torch.no_grad()")
        for o, t in zip(out, (q, k)):
            if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device or _heads(o) is not o:
                raise ValueError(f"out must hold {t.dtype} tensors of q's and k's shapes on {t.device}, "
                                 "their last dim contiguous and rows at 16-byte steps")
        _check_overlap(q, k, out)
    if grad:
        res = _QKNormRope.apply(q, k, pos, rotary, q_weight, k_weight, eps, rows, dev)
        _lib.mark_leaves(dev, res[0].grad_fn)
        return res
    res = _forward(q, k, pos, rotary, q_weight, k_weight, eps, rows, dev, out)
    if out is not None:
        torch.autograd.graph.increment_version(out)      # a graph that saved them must notice
    return res


def _span(t: torch.Tensor):
    """First byte and the byte behind the last that `t` reaches."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def folded(t: torch.Tensor) -> bool:
    """Whether two elements of `t` may lie in one place."""
    extent = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < extent:
            return True
        extent += s * (n - 1)
    return False


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (rows, heads, dim) or (batch, heads, rows, dim) tensors may
    share memory.  Slices of one buffer interleave (q and k of a fused
    projection): those are apart where all rows of both start a step's multiple
    away from each other and the heads of each have columns of their own within
    the step."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    step = 0
    for t in (a, b):
        for d in range(t.dim() - 1):
            if d != 1 and t.shape[d] > 1:             # rows and batches
                step = math.gcd(step, t.stride(d) * t.element_size())
    la, lb = (_span(t[:1] if t.dim() == 3 else t[:1, :, :1])[1] - t.data_ptr() for t in (a, b))
    off = (b0 - a0) % step if step else 0
    return off < la or off + lb > step


def _check_overlap(q, k, out):
    """In place means exactly in place."""
    def same(a, b):
        return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()

    qo, ko = out
    for o in out:
        if folded(o):
            raise ValueError("out must not be a broadcast view, nor overlap itself otherwise")
    if overlap(qo, ko) or overlap(qo, k) or overlap(ko, q) or not (same(qo, q) or not overlap(qo, q)) or \
            not (same(ko, k) or not overlap(ko, k)):
        raise ValueError("out may be q and k themselves, but must not overlap them otherwise")
