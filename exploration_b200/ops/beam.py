"""Beam search over a paged cache: the selection and the reordering that follows it.

* :func:`beam_select` takes the best ``beams`` continuations of every group
  from the step's logits, in one pass over them.
* :func:`beam_reorder` makes the cache follow the selection: new page tables,
  and a copy of the partly filled page for each beam that takes over another
  beam's state. All beams of a group have the same length; a page being filled
  belongs to one beam, full pages are shared and never written again; every
  beam holds one spare page.

Both are for inference. CUDA tensors run the sm_100a kernels of ``csrc/beam``
(the extension makes the checks that the functions here make for CPU tensors);
CPU tensors run the definitions below.
"""
from __future__ import annotations

import torch

from . import _native
from .gated_reference import NEG_INF, work_dtype
from .launch import count

MAX_BEAMS = 32


def beam_select(logits, scores, finished, eos):
    """Best continuations of each group: ``(scores, parents, tokens, finished)``, all ``[groups, beams]``.

    ``logits [groups, beams, vocab]``, cumulative log-probabilities ``scores
    [groups, beams]`` (fp32) and ``finished`` (bool). A running beam offers
    token ``t`` at ``score + (logit_t - logsumexp(logits))``; a finished one
    offers only ``(eos, score)``. Candidates are ordered inside a beam by logit,
    then token, and across beams by score (fp32), then beam, best first. A
    beam whose logsumexp is not finite offers tokens ``0, 1, ...`` at ``-inf``. ``parents`` and
    ``tokens`` are int64; ``finished`` is true for an ended parent or token
    ``eos`` (``-1``: no token ends a beam).
    """
    if logits.is_cuda:
        out = _native.native(logits).beam_select(logits, scores, finished, eos)
        count("beam_select", ("dtype", "beams"), (logits.dtype, logits.shape[1]))
        return out
    if logits.ndim != 3 or scores.shape != logits.shape[:2] or finished.shape != scores.shape:
        raise ValueError("expected logits [groups, beams, vocab] and scores, finished [groups, beams]")
    if scores.dtype != torch.float32 or finished.dtype != torch.bool:
        raise ValueError("scores must be fp32 and finished bool")
    if not (logits.device == scores.device == finished.device):
        raise ValueError("all tensors must be on one device")
    if not 1 <= logits.shape[1] <= MAX_BEAMS or logits.shape[2] < 1:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams and at least one token")
    if _native.wants_grad(logits, scores):
        raise ValueError("beam_select is for inference: it has no gradient")
    eos = int(eos)
    if not -1 <= eos < logits.shape[2]:
        raise ValueError("eos must be a token or -1")
    return select_reference(logits, scores, finished, eos)


def beam_reorder(k_cache, v_cache, tables, spare, parents, lengths):
    """The cache's ``(tables, spare)`` after beam ``i`` of each group took over ``parents[g, i]``.

    Pools ``[layers, pages, kv_heads, page, head_dim]``; ``tables [groups,
    beams, width]`` and ``spare [groups, beams]`` (int32); ``parents [groups,
    beams]`` (int64); ``lengths [groups]`` (int32): tokens of each of the
    group's beams. The first ``lengths % page`` rows of a parent's page being
    filled are copied into the spare page of each beam whose parent is another
    beam; that page takes its place in the new table and the old one becomes
    the spare. The given tables are left as they are. Pools without an element (no
    layers, say) give the tables and copy nothing.
    """
    if k_cache.is_cuda:
        out = _native.native(k_cache).beam_reorder(k_cache, v_cache, tables, spare, parents, lengths)
        count("beam_reorder", ("dtype", "page"), (k_cache.dtype, k_cache.shape[3]))
        return out
    if k_cache.ndim != 5 or k_cache.shape != v_cache.shape or tables.ndim != 3 or spare.shape != tables.shape[:2] \
            or parents.shape != spare.shape or lengths.shape != spare.shape[:1] or tables.shape[2] < 1:
        raise ValueError("expected pools [layers, pages, kv_heads, page, head_dim], tables [groups, beams, width], "
                         "spare, parents [groups, beams] and lengths [groups]")
    if k_cache.shape[3] < 1:
        raise ValueError("a page must hold at least one token")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype.itemsize % 2:
        raise ValueError("key and value pools must have one dtype of 16 bits or more")
    if tables.dtype != torch.int32 or spare.dtype != torch.int32 or lengths.dtype != torch.int32 \
            or parents.dtype != torch.int64:
        raise ValueError("tables, spare and lengths must be int32 and parents int64")
    if not (k_cache.device == v_cache.device == tables.device == spare.device == parents.device == lengths.device):
        raise ValueError("all tensors must be on one device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("cache pools must be contiguous")
    if _native.wants_grad(k_cache, v_cache):
        raise ValueError("beam_reorder is for inference: it has no gradient")
    return reorder_reference(k_cache, v_cache, tables, spare, parents, lengths)


# ----------------------------------------------------------------------------
# definitions (CPU path and oracle)
# ----------------------------------------------------------------------------

def select_reference(logits, scores, finished, eos):
    groups, beams, vocab = logits.shape
    keep = min(beams, vocab)
    x = logits.to(work_dtype(logits))
    # x - logsumexp(x) from the distance to the largest logit: nothing is lost to the logits' size.
    peak = x.amax(-1, keepdim=True)
    log_sum = (x - peak).exp().sum(-1, keepdim=True).log()
    alive = torch.isfinite(peak) & torch.isfinite(log_sum)
    best, token = x.sort(dim=-1, descending=True, stable=True)
    best, token = best[..., :keep], token[..., :keep]
    total = scores[..., None] + ((best - peak) - log_sum).float()
    rank = torch.arange(keep, device=logits.device)
    total = torch.where(alive & ~total.isnan(), total, NEG_INF)
    token = torch.where(alive, token, rank)
    first = rank == 0
    ended = finished[..., None]
    total = torch.where(ended, torch.where(first, scores[..., None], NEG_INF), total)
    token = torch.where(ended, eos, token)
    total, order = total.flatten(1).sort(dim=-1, descending=True, stable=True)
    total, order = total[:, :beams], order[:, :beams]
    parents, tokens = order // keep, token.flatten(1).gather(1, order)
    return total.contiguous(), parents, tokens, finished.gather(1, parents) | (tokens == eos)


def reorder_reference(k_cache, v_cache, tables, spare, parents, lengths):
    page = k_cache.shape[3]
    fresh, freed = tables.clone(), spare.clone()
    for g in range(tables.shape[0]):
        tail, rows = divmod(max(0, int(lengths[g])), page)
        for beam in range(tables.shape[1]):
            parent = int(parents[g, beam])
            if parent == beam or not 0 <= parent < tables.shape[1]:
                continue
            fresh[g, beam, :tail] = tables[g, parent, :tail]
            if rows and tail < tables.shape[2]:
                source, target = int(tables[g, parent, tail]), int(spare[g, beam])
                k_cache[:, target, :, :rows] = k_cache[:, source, :, :rows]
                v_cache[:, target, :, :rows] = v_cache[:, source, :, :rows]
                fresh[g, beam, tail], freed[g, beam] = target, tables[g, beam, tail]
    return fresh, freed
