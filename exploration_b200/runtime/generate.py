"""Incremental generation with :class:`BaselineModel`: paged cache, greedy and beam search.

The prompt is encoded in chunks (:func:`paged_append`, :func:`paged_attention`
in every layer), then every step runs one token a beam, takes the best
continuations (:func:`beam_select`) and lets the cache follow them
(:func:`beam_reorder`). Lengths, positions, tables and the selection stay on
the device; the host looks at them only to stop early, and at the end for
kernels that gave up a wait.
"""
from __future__ import annotations

import torch

from ..ops import _native, fused
from ..ops.beam import MAX_BEAMS, beam_reorder, beam_select
from ..ops.paged import MIN_PAGE

STOP_EVERY = 16      # steps between looks at whether every beam has ended


def check_waits(device):
    """Raises when a kernel on ``device`` gave up a bounded wait: what it should have written is undefined."""
    if device.type != "cuda":
        return
    torch.cuda.current_stream(device).synchronize()
    site, cta = _native.load().device_errors(device.index)
    if site:
        raise RuntimeError(f"a kernel on {device} gave up a wait (site {site}, CTA {cta}): its results are undefined")


class PagedCache:
    """Key/value pools of all layers, and the page tables of groups of beams.

    ``lengths`` are the prompts' lengths. The beams of a group share the
    prompt's full pages; from the page being filled on, each beam has pages of
    its own and one spare page (see :func:`beam_reorder`).
    """

    def __init__(self, layers, kv_heads, head_dim, lengths, new_tokens, *, beams=1, page=64, dtype=torch.float32,
                 device="cpu"):
        if not lengths or min(lengths) < 1 or new_tokens < 0:
            raise ValueError("prompts must hold at least one token")
        if page < MIN_PAGE or page & (page - 1):
            raise ValueError(f"page must be a power of two of at least {MIN_PAGE}")
        self.page, self.beams = page, beams
        width = -(-(max(lengths) + new_tokens) // page)
        tables = torch.zeros(len(lengths), beams, width, dtype=torch.int32)
        spare = torch.zeros(len(lengths), beams, dtype=torch.int32)
        at = 0
        for g, n in enumerate(lengths):
            shared, need = n // page, -(-(n + new_tokens) // page)
            tables[g, :, :shared] = torch.arange(at, at + shared, dtype=torch.int32)
            at += shared
            for b in range(beams):
                tables[g, b, shared:need] = torch.arange(at, at + need - shared, dtype=torch.int32)
                spare[g, b] = at + need - shared
                at += need - shared + 1
        self.tables, self.spare = tables.to(device), spare.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        shape = (layers, at, kv_heads, page, head_dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))

    @property
    def rows(self):
        """Tables of every beam, ``[groups * beams, width]``."""
        return self.tables.flatten(0, 1)

    def reorder(self, parents):
        self.tables, self.spare = beam_reorder(self.k, self.v, self.tables, self.spare, parents, self.lengths)


def _check(model, prompts, max_new_tokens, beams, eos, prefill_chunk):
    if not hasattr(model, "decode"):
        raise ValueError("generation needs a model with incremental decoding (BaselineModel)")
    if not prompts or max_new_tokens < 1 or prefill_chunk < 1:
        raise ValueError("generation needs prompts, a positive number of new tokens and a positive chunk")
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams")
    vocab = model.embedding.weight.shape[0]
    if eos is not None and not 0 <= eos < vocab:
        raise ValueError("eos must be a token")


@torch.no_grad()
def generate(model, prompts, max_new_tokens, *, beams=1, eos=None, page=64, prefill_chunk=4096):
    """Best continuations of every prompt: ``(tokens [prompts, beams, n], scores [prompts, beams])``.

    ``prompts`` is a list of token lists (or 1-D tensors) of any lengths;
    ``beams=1`` is greedy decoding. ``scores`` are cumulative log-probabilities,
    best first; a hypothesis that ended is padded with ``eos``. ``n`` is at most
    ``max_new_tokens`` (less when every beam has ended). On a GPU the call waits
    for its result and raises ``RuntimeError`` when a kernel gave up a wait.
    """
    _check(model, prompts, max_new_tokens, beams, eos, prefill_chunk)
    device = model.embedding.weight.device
    prompts = [torch.as_tensor(p, dtype=torch.long).reshape(-1) for p in prompts]
    lengths = [len(p) for p in prompts]
    groups, longest = len(prompts), max(lengths)
    dtype = fused.compute_dtype(model.embedding.weight, model.embedding.weight.dtype)
    cache = PagedCache(len(model.blocks), model.heads, model.hd, lengths, max_new_tokens, beams=beams, page=page,
                       dtype=dtype, device=device)
    ids = torch.zeros(groups, longest, dtype=torch.long)
    positions = torch.full((groups, longest), -1, dtype=torch.int32)
    for g, p in enumerate(prompts):
        ids[g, :len(p)] = p
        positions[g, :len(p)] = torch.arange(len(p), dtype=torch.int32)
    if bool(((ids < 0) | (ids >= model.embedding.weight.shape[0])).any()):
        raise ValueError("prompt tokens must lie in the model's vocabulary")     # on a GPU a fault of its embedding
    ids, positions = ids.to(device), positions.to(device)
    cos, sin = model.rope.tables(torch.arange(longest + max_new_tokens, device=device))

    def run(tokens, at, tables):
        return model.decode(tokens, cache.k, cache.v, cos, sin, tables, at)

    # Prompts: the first beam of each group; its state then fans out to the others.
    last = (cache.lengths.long() - 1)[:, None, None]
    final = None
    first_rows = cache.tables[:, 0].contiguous()
    for lo in range(0, longest, prefill_chunk):
        hi = min(lo + prefill_chunk, longest)
        x = run(ids[:, lo:hi], positions[:, lo:hi].contiguous(), first_rows)
        picked = x.gather(1, (last - lo).clamp(0, hi - lo - 1).expand(-1, 1, x.shape[-1]))
        inside = (last >= lo) & (last < hi)
        final = picked if final is None else torch.where(inside, picked, final)
    cache.reorder(torch.zeros(groups, beams, dtype=torch.int64, device=device))
    logits = model.logits(final).expand(-1, beams, -1)
    scores = torch.full((groups, beams), float("-inf"), device=device)
    scores[:, 0] = 0.0
    finished = torch.zeros(groups, beams, dtype=torch.bool, device=device)
    end = -1 if eos is None else int(eos)
    out = torch.zeros(groups, beams, max_new_tokens, dtype=torch.int64, device=device)
    for step in range(max_new_tokens):
        scores, parents, tokens, finished = beam_select(logits, scores, finished, end)
        if beams > 1:
            out = out.gather(1, parents[..., None].expand_as(out))
        out[:, :, step] = tokens
        if step + 1 == max_new_tokens:
            break
        if eos is not None and step % STOP_EVERY == STOP_EVERY - 1 and bool(finished.all()):
            out = out[:, :, :step + 1]
            break
        if beams > 1:
            cache.reorder(parents)
        at = cache.lengths[:, None].expand(groups, beams).reshape(-1, 1)
        x = run(tokens.reshape(-1, 1), at, cache.rows)
        cache.lengths += 1
        logits = model.logits(x).view(groups, beams, -1)
    check_waits(device)
    return out, scores
