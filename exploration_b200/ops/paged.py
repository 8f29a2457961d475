"""Attention of a dense causal model over a paged key/value cache.

A cache is two pools ``[pages, kv_heads, page, head_dim]`` (keys, values) and
tables ``[batch, width]`` (int32): ``tables[b, j]`` names the pool page with
positions ``[j * page, (j + 1) * page)`` of sequence ``b``. ``page`` is a power
of two of at least 16. New tokens come with ``positions [batch, tokens]``
(int32; int64 is converted), ``-1`` marking a padding row, whose output is
zero. Everything that says how long a sequence is lies on the device, so
one captured CUDA graph of a step serves every later step.

* :func:`paged_append` rotates queries and keys (split-half RoPE from fp32
  tables) and writes keys and values into their pages;
* :func:`paged_attention` reads keys ``0 .. position`` for every row. Query
  heads ``h * g .. h * g + g - 1`` share key head ``h``.

Both are for inference: they have no gradient and refuse inputs that need
one. CUDA tensors (fp32, fp16, bf16) run the sm_100a kernels of
``csrc/paged``; CPU tensors run the definitions below. Rows of the cache past
a sequence's largest position may hold anything (a non-finite key or value that
one row of a call sees may reach the call's other rows of that sequence). A position past the end of
the table (or of the rotation tables) or a table entry outside the pool is
the caller's error: CUDA kernels stay inside the buffers, what such rows
read or lose is undefined.
"""
from __future__ import annotations

import math

import torch

from . import _native
from .gated_reference import NEG_INF, work_dtype
from .launch import count

MIN_PAGE = 16
MAX_HEAD_DIM = 256


def _check_cache(x, k_cache, v_cache, tables, positions):
    """Checks shared by the two operators; ``x [batch, tokens, heads, head_dim]``.

    The extension makes the same ones (and that CUDA pools are contiguous and of
    a native dtype) for CUDA tensors, where a call takes a few microseconds.
    """
    if x.ndim != 4 or k_cache.ndim != 4 or k_cache.shape != v_cache.shape or x.shape[3] != k_cache.shape[3]:
        raise ValueError("expected rows [batch, tokens, heads, head_dim] and caches [pages, kv_heads, page, head_dim]")
    page, dim = k_cache.shape[2], k_cache.shape[3]
    if page < MIN_PAGE or page & (page - 1):
        raise ValueError(f"page must be a power of two of at least {MIN_PAGE}")
    if dim % 2 or not 2 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be even and at most {MAX_HEAD_DIM}")
    if k_cache.shape[1] < 1 or x.shape[2] < 1 or x.shape[2] % k_cache.shape[1]:
        raise ValueError("query heads must be a positive multiple of the cache's heads")
    if positions.shape != x.shape[:2] or tables.ndim != 2 or tables.shape[0] != x.shape[0]:
        raise ValueError("expected positions [batch, tokens] and tables [batch, width]")
    if positions.dtype not in (torch.int32, torch.int64) or tables.dtype != torch.int32:
        raise ValueError("positions must be int32 or int64 and tables int32")
    if x.dtype != k_cache.dtype or x.dtype != v_cache.dtype:
        raise ValueError("rows and caches must have one dtype")
    device = x.device
    if not (k_cache.device == v_cache.device == tables.device == positions.device == device):
        raise ValueError("all tensors must be on one device")
    if _native.wants_grad(x, k_cache, v_cache):
        raise ValueError("paged operators are for inference: they have no gradient")


def paged_append(q, k, v, cos, sin, k_cache, v_cache, tables, positions):
    """Write the new tokens' keys (rotated) and values into the cache; returns the rotated queries.

    ``q [batch, tokens, heads, head_dim]`` and ``k, v [batch, tokens, kv_heads,
    head_dim]`` may be strided views of one projection. ``cos, sin [positions,
    head_dim / 2]`` are fp32 (``RotaryEmbedding.tables``). The caches are
    updated in place; rows at position ``-1`` write nothing and give zeros.
    """
    if q.is_cuda:
        out = _native.native(q).paged_append(q, k, v, cos, sin, k_cache, v_cache, tables, positions)
        count("paged_append", ("dtype", "head_dim", "page"), (q.dtype, q.shape[3], k_cache.shape[2]))
        return out
    _check_cache(q, k_cache, v_cache, tables, positions)
    if k.shape != v.shape or k.shape != (*q.shape[:2], k_cache.shape[1], q.shape[3]):
        raise ValueError("expected k, v [batch, tokens, kv_heads, head_dim]")
    if k.dtype != q.dtype or v.dtype != q.dtype or not (k.device == v.device == cos.device == sin.device == q.device):
        raise ValueError("queries, keys, values and rotation tables must match in dtype and device")
    if cos.shape != sin.shape or cos.ndim != 2 or cos.shape[1] * 2 != q.shape[3] \
            or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("expected fp32 cos, sin [positions, head_dim / 2]")
    if _native.wants_grad(k, v, cos, sin):
        raise ValueError("paged operators are for inference: they have no gradient")
    return append_reference(q, k, v, cos, sin, k_cache, v_cache, tables, positions)


def paged_attention(q, k_cache, v_cache, tables, positions):
    """``softmax(q . k / sqrt(head_dim)) v`` over keys ``0 .. position`` of each row's sequence.

    ``q [batch, tokens, heads, head_dim]``; the result has its shape and dtype.
    """
    if q.is_cuda:
        ext = _native.native(q)
        out = ext.paged_attention(q, k_cache, v_cache, tables, positions)
        count("paged_attention", ("dtype", "head_dim", "page", "path"),
              (q.dtype, q.shape[3], k_cache.shape[2], ext.paged_attention_path(q, k_cache, v_cache)))
        return out
    _check_cache(q, k_cache, v_cache, tables, positions)
    return attention_reference(q, k_cache, v_cache, tables, positions)


# ----------------------------------------------------------------------------
# definitions (CPU path and oracle)
# ----------------------------------------------------------------------------

def rotate_reference(x, cos, sin):
    """Split-half rotation of ``x [..., heads, head_dim]`` by ``cos, sin [..., head_dim / 2]``."""
    dtype = work_dtype(x)
    first, second = x.to(dtype).chunk(2, -1)
    cos, sin = cos[..., None, :].to(dtype), sin[..., None, :].to(dtype)
    return torch.cat((first * cos - second * sin, second * cos + first * sin), -1).to(x.dtype)


def append_reference(q, k, v, cos, sin, k_cache, v_cache, tables, positions):
    page = k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    batch, token = (positions >= 0).nonzero(as_tuple=True)
    at = positions[batch, token].long()
    pages = tables[batch, at // page].long()
    out[batch, token] = rotate_reference(q[batch, token], cos[at], sin[at])
    k_cache[pages, :, at % page] = rotate_reference(k[batch, token], cos[at], sin[at])
    v_cache[pages, :, at % page] = v[batch, token]
    return out


def attention_reference(q, k_cache, v_cache, tables, positions):
    dtype = work_dtype(q)
    group, page = q.shape[2] // k_cache.shape[1], k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    for b in range(q.shape[0]):
        rows = positions[b] >= 0
        if not bool(rows.any()):
            continue
        pos = positions[b, rows].long()
        n = int(pos.max()) + 1
        pages = tables[b, :-(-n // page)].long()
        # [kv_heads, n, head_dim] -> [heads, n, head_dim]
        k, v = (c[pages].transpose(0, 1).flatten(1, 2)[:, :n].to(dtype).repeat_interleave(group, 0)
                for c in (k_cache, v_cache))
        logits = q[b, rows].transpose(0, 1).to(dtype) @ k.transpose(1, 2) / math.sqrt(q.shape[3])
        hidden = torch.arange(n, device=q.device) > pos[:, None]
        out[b, rows] = (logits.masked_fill(hidden, NEG_INF).softmax(-1) @ v).transpose(0, 1).to(q.dtype)
    return out
