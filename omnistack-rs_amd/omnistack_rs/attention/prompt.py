"""Attention of whole prompts packed one after another (omni_prompt_attn).

The prompt's own step before its keys and values go into the packed cache
(``PackedKVEncoder`` / ``PagedKVCache``, which ``omni_attn`` and
``paged_attention`` then read): 16-bit q, k, v as the projections and
``kernels.rope.qk_norm_rope`` leave them, sequences of different lengths in
one batch without padding, grouped heads, causal or not, with a gradient (to
train query adapters through).  ``reference_attn`` is the padded fp32
counterpart.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib
from ..kernels.rope import folded, overlap

_HEAD_DIMS = (32, 64, 128)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as the kernels read it: the last dim contiguous, 16-byte steps, no
    huge token stride."""
    if t.data_ptr() % 16 == 0 and t.stride(0) < 1 << 24:
        if t.is_contiguous():
            return t
        a, b, c = t.stride()
        if c == 1 and (a % 8 == 0 or t.shape[0] == 1) and (b % 8 == 0 or t.shape[1] == 1):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    s = t.stride()
    return _lib.I64x2(0 if t.shape[0] == 1 else s[0], 0 if t.shape[1] == 1 else s[1])


def _check(q, k, v, cu_seqlens, scale, validate):
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"q must be (N, n_heads, head_dim), k and v (N, n_kv_heads, head_dim), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    N, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape[0] != N or k.shape[2] != D or Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} disagree (n_heads a multiple of n_kv_heads)")
    if D not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {D}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must share float16 or bfloat16 (float32: reference_attn), got {q.dtype}, {k.dtype} "
                         f"and {v.dtype}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not abs(scale) <= 2.3e38:                     # the kernels multiply it by log2 e
        raise ValueError(f"scale must be finite and at most 2.3e38 in size, got {scale}")
    cu = cu_seqlens if isinstance(cu_seqlens, torch.Tensor) else torch.as_tensor(cu_seqlens)
    if cu.dim() != 1 or cu.numel() < 1 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cu_seqlens must be int32 or int64 (n_sequences + 1,), got {cu.dtype} {tuple(cu.shape)}")
    if validate or not cu.is_cuda:
        host = cu.cpu().to(torch.int64)
        if int(host[0]) != 0 or bool((host[1:] < host[:-1]).any()) or int(host[-1]) > N:
            raise ValueError(f"cu_seqlens must rise from 0 to at most {N}")
    dev = _lib.require_device(q, k, v, cu if cu.is_cuda else None)
    if cu.dtype != torch.int32 or not cu.is_cuda or not cu.is_contiguous():
        cu = cu.to(device=dev, dtype=torch.int32).contiguous()
    return dev, cu, scale


def _forward(q, k, v, cu, scale, causal, out, need_lse, dev, need_rest=False):
    N, Hq, D = q.shape
    qc, kc, vc = _rows(q), _rows(k), _rows(v)
    o = _lib.empty_as(q) if out is None else out
    lse = None
    if need_lse:                                     # the kernel leaves rows of no sequence as they were where out= does
        lse = torch.empty(Hq, N, dtype=torch.float32, device=dev)
        if out is not None:
            lse.fill_(-math.inf)
    rest = _lib.empty_as(q) if need_rest else None
    rc = _lib.on_device(
        dev, _lib.lib().omni_prompt_attn, qc.data_ptr(), _strides(qc), kc.data_ptr(), _strides(kc), vc.data_ptr(),
        _strides(vc), _lib.dtype_code(q.dtype), N, Hq, k.shape[1], D, cu.data_ptr(), cu.numel() - 1, scale, int(causal),
        int(out is None), o.data_ptr(), _strides(o), _lib.ptr(lse), _lib.ptr(rest), _strides(rest) if need_rest else None,
        _lib.stream_of(dev))
    if rc:
        _lib.check(rc)
    return (o, lse, rest) if need_rest else (o, lse)


class _PromptAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, scale, causal, dev):
        q, k, v = _rows(q), _rows(k), _rows(v)
        o, lse, rest = _forward(q, k, v, cu, scale, causal, None, True, dev, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, cu)
        ctx.scale, ctx.causal, ctx.dev = scale, causal, dev
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, _):
        _lib.refuse_tangents("prompt_attention's gradient", do)
        q, k, v, o, rest, lse, cu = ctx.saved_tensors
        N, Hq, D = q.shape
        do = _rows(do)
        dq, dk, dv = (_lib.empty_as(t) for t in (q, k, v))
        L = _lib.lib()
        ws_bytes = _lib.on_device(ctx.dev, L.omni_prompt_attn_backward_workspace_size, N, Hq, k.shape[1], D, cu.numel() - 1)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=ctx.dev) if ws_bytes else None
        _lib.check(_lib.on_device(
            ctx.dev, L.omni_prompt_attn_backward, q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(),
            _strides(v), _lib.dtype_code(q.dtype), N, Hq, k.shape[1], D, cu.data_ptr(), cu.numel() - 1, ctx.scale,
            int(ctx.causal), o.data_ptr(), _strides(o), rest.data_ptr(), _strides(rest), lse.data_ptr(),
            do.data_ptr(), _strides(do), dq.data_ptr(), _strides(dq), dk.data_ptr(), _strides(dk), dv.data_ptr(),
            _strides(dv), _lib.ptr(ws), ws_bytes, _lib.stream_of(ctx.dev)))
        return dq, dk, dv, None, None, None, None


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens, *, causal: bool = True,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                     validate: bool = True):
    """softmax(scale q k^T) v within each packed sequence.

    q (N, n_heads, head_dim), k and v (N, n_kv_heads, head_dim): float16 or
    bfloat16, head_dim 32, 64 or 128, any strides (slices of a fused projection
    are read in place). ``cu_seqlens`` (n_sequences + 1,): where each sequence
    starts and the last one ends, int32 or int64 on the device or on the host;
    lengths of zero are fine. ``causal``: token t sees tokens up to t of its
    sequence. Returns (N, n_heads, head_dim) in q's dtype, and with
    ``return_lse`` the rows' log of summed exponentials, float32 (n_heads, N;
    it has no gradient). Scores are fp32 numbers: one of size X is off by about
    2^-24 X, and the gradient's probabilities by as much of themselves; past
    2^23 gradients have no meaning and outputs may not be finite. Gradients for
    q, k and v, once and in reverse mode (dual tensors are refused), all three
    whichever are asked for; forward and backward can be captured in a HIP
    graph (``validate`` off, cu_seqlens on the device) once no eager autograd
    graph of the same leaves is alive: one through these operators on the
    default stream is refused, as is one of leaves passed to them directly.
    Rows behind the last sequence are zeros (lse -inf); in ``out``, a tensor to
    write into (no gradient then), they stay as they were. ``validate`` checks
    cu_seqlens on the host: a device sync when it is on the device, some 25 us
    a call. (On the host it is always checked, and copied to the device.)
    Without it values that break the rules give rows of no meaning."""
    _lib.refuse_tangents("prompt_attention", q, k, v, out)
    dev, cu, scale = _check(q, k, v, cu_seqlens, scale, validate)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if out is not None:
        if grad or torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("out= takes no gradient: call it under torch.no_grad()")
        if out.shape != q.shape or out.dtype != q.dtype or out.device != dev or _rows(out) is not out:
            raise ValueError(f"out must be a {q.dtype} tensor of shape {tuple(q.shape)} on {dev}, its last dim contiguous "
                             "and rows at 16-byte steps")
        if folded(out) or any(overlap(out, t) for t in (q, k, v)):
            raise ValueError("out must not overlap q, k or v, nor itself")
    if grad:
        o, lse = _PromptAttention.apply(q, k, v, cu, scale, causal, dev)
        _lib.mark_leaves(dev, o.grad_fn)
        return (o, lse) if return_lse else o
    o, lse = _forward(q, k, v, cu, scale, causal, out, return_lse, dev)
    if out is not None:
        torch.autograd.graph.increment_version(out)      # a graph that saved it must notice
    return (o, lse) if return_lse else o
