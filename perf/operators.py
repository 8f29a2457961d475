"""Cases of the paged-cache decoding operators, their plain forms and their definitions in 64 bits.

The operators: ``paged_append`` (rotate queries and keys, write keys and values into the pages),
``paged_attention`` (new tokens over the cache), ``beam_select`` (best continuations of every group of
beams) and ``beam_reorder`` (the cache's tables and partly filled pages after a selection).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EOS = 1


def listed():
    return [
        # One new token for each of a batch of running sequences, once a layer: launch latency.
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 32, "new": 1, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 64, "low": 3, "high": 500},
        # A chunk of four prompts of different lengths, shared key heads: copy bandwidth.
        {"name": "append_chunk", "op": "append", "dtype": "bf16", "batch": 4, "new": 2011, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "low": 2100, "high": 3011},
        # A short conversation on the small model (4 heads of 64): latency of a single step.
        {"name": "step_short", "op": "attention", "dtype": "bf16", "batch": 4, "new": 1, "ragged": False,
         "heads": 4, "kv_heads": 4, "dim": 64, "page": 16, "low": 1, "high": 517},
        # A serving batch of very different lengths with shared key heads: the cache is read once a step.
        {"name": "step_batch", "op": "attention", "dtype": "bf16", "batch": 64, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "low": 17, "high": 16384},
        # Two long documents in full precision: few rows, a long axis.
        {"name": "step_long_fp32", "op": "attention", "dtype": "fp32", "batch": 2, "new": 1, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 128, "low": 60001, "high": 60001},
        # A few drafted tokens a sequence, checked in one call.
        {"name": "verify_few", "op": "attention", "dtype": "fp16", "batch": 16, "new": 5, "ragged": True,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 32, "low": 700, "high": 4099},
        # A late chunk of a 64k-token prompt (16 heads of 64): arithmetic.
        {"name": "chunk_long", "op": "attention", "dtype": "bf16", "batch": 1, "new": 2048, "ragged": False,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 64, "low": 65536, "high": 65536},
        # Prompt chunks of different lengths side by side, one sequence without any new token.
        {"name": "chunk_ragged", "op": "attention", "dtype": "fp16", "batch": 6, "new": 1111, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "low": 1500, "high": 8191},
        # Four searches of width four over a byte vocabulary: latency of a step.
        {"name": "select_bytes", "op": "select", "dtype": "fp32", "groups": 4, "beams": 4, "vocab": 256,
         "masked": False},
        # A batch of searches over a large vocabulary of odd size, part of it masked: one pass over the logits.
        {"name": "select_words", "op": "select", "dtype": "bf16", "groups": 8, "beams": 8, "vocab": 100003,
         "masked": True},
        # The small model's cache (3 layers) after a step of width four.
        {"name": "reorder_short", "op": "reorder", "dtype": "bf16", "layers": 3, "groups": 4, "beams": 4,
         "kv_heads": 4, "dim": 64, "page": 16, "low": 5, "high": 61},
        # A 12-layer cache with 16 heads: partly filled pages of all layers are copied.
        {"name": "reorder_deep", "op": "reorder", "dtype": "bf16", "layers": 12, "groups": 4, "beams": 6,
         "kv_heads": 16, "dim": 64, "page": 64, "low": 90, "high": 127},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "attention", "select", "reorder"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "append":
        heads, kv = rng.choice(((4, 4), (16, 16), (24, 24), (32, 8), (12, 4)))
        dim, new = rng.choice((64, 128)), _spread(rng, 1, 2000)
        batch = _spread(rng, 1, max(1, min(64, 8000 // new)))
        low = new + rng.randint(0, 100)
        return {"op": op, "dtype": dtype, "batch": batch, "new": new, "ragged": rng.random() < 0.5, "heads": heads,
                "kv_heads": kv, "dim": dim, "page": rng.choice((16, 32, 64, 128)), "low": low,
                "high": low + rng.randint(0, 400)}
    if op == "attention":
        heads, kv = rng.choice(((4, 4), (16, 16), (24, 24), (32, 8), (16, 2), (12, 4)))
        dim = rng.choice((64, 128))
        new = rng.choice((1, 1, _spread(rng, 2, 16), _spread(rng, 17, 2048)))
        if dtype == "fp32":
            new = min(new, 64)
        # Bounded by the largest listed case: its arithmetic and the bytes of the longest step.
        top = min(65536, int(5e11 / (4 * dim * heads * new)))
        high = _spread(rng, new, max(new, top))
        batch = _spread(rng, 1, max(1, min(64, int(2e9 / (4 * high * kv * dim * BYTES[dtype])),
                                           int(5e11 / (4.0 * dim * heads * new * high)))))
        return {"op": op, "dtype": dtype, "batch": batch, "new": new, "ragged": new > 1 and rng.random() < 0.5,
                "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice((16, 32, 64, 128)),
                "low": rng.randint(new, high), "high": high}
    if op == "select":
        beams, vocab = rng.choice((1, 2, 3, 4, 5, 8)), _spread(rng, 128, 100003)
        return {"op": op, "dtype": dtype, "groups": _spread(rng, 1, 8), "beams": beams, "vocab": vocab,
                "masked": rng.random() < 0.5}
    page = rng.choice((16, 32, 64))
    low = rng.randint(1, 2 * page - 1)
    return {"op": op, "dtype": rng.choice(("bf16", "fp16")), "layers": _spread(rng, 1, 12),
            "groups": _spread(rng, 1, 4), "beams": rng.choice((1, 2, 3, 4, 6)), "kv_heads": rng.choice((4, 8, 16)),
            "dim": 64, "page": page, "low": low, "high": rng.randint(low, 2 * page - 1)}


# ----------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------

def _lengths(count, low, high):
    """Lengths spread evenly over [low, high], long and short ones mixed."""
    if count == 1:
        return [high]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, count) == 1)
    return [low + (high - low) * ((i * step + count - 1) % count) // (count - 1) for i in range(count)]


def _counts(case):
    """New tokens of each sequence; a ragged chunk of several sequences has an empty one."""
    batch, new = case["batch"], case["new"]
    if not case["ragged"]:
        return [new] * batch
    counts = [max(1, c) for c in _lengths(batch, max(1, new // 3), new)]
    if batch > 2:
        counts[batch // 2] = 0
    return counts


def _paged(case, gen, dtype, layers=None, extra=0):
    """Pools with the pages of all sequences in random order, and the tables."""
    lengths = _lengths(case["batch"], case["low"], case["high"])
    page, width = case["page"], -(-max(lengths) // case["page"])
    needed = [-(-n // page) for n in lengths]
    shape = (sum(needed) + extra, case["kv_heads"], page, case["dim"])
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    order = torch.randperm(sum(needed), generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for row, count in enumerate(needed):
        tables[row, :count] = order[at:at + count]
        at += count
    return lengths, k, v, tables


def _positions(case, lengths):
    rows = torch.full((case["batch"], case["new"]), -1, dtype=torch.int32)
    for row, (n, count) in enumerate(zip(lengths, _counts(case))):
        rows[row, :count] = torch.arange(n - count, n)
    return rows.cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    state = {"case": case}
    if op in ("append", "attention"):
        lengths, k_cache, v_cache, tables = _paged(case, gen, dtype)
        batch, new, heads, kv, dim = (case[x] for x in ("batch", "new", "heads", "kv_heads", "dim"))
        state.update(lengths=lengths, counts=_counts(case), k_cache=k_cache, v_cache=v_cache, tables=tables,
                     positions=_positions(case, lengths))
        if op == "append":
            # The projection's output: queries, keys and values side by side for each token.
            state["qkv"] = torch.randn((batch, new, heads + 2 * kv, dim), generator=gen, device="cuda", dtype=dtype)
            index = torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None]
            rate = 10_000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
            state["cos"], state["sin"] = (index * rate).cos().float(), (index * rate).sin().float()
        else:
            # Logits with a standard deviation of two: some keys carry most of the weight.
            state["q"] = (2 * torch.randn((batch, new, heads, dim), generator=gen, device="cuda")).to(dtype)
        return state
    if op == "select":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        # A peaked distribution; hypotheses a few nats apart, best first; some of them ended.
        state["logits"] = (3 * torch.randn((groups, beams, vocab), generator=gen, device="cuda")).to(dtype)
        if case["masked"]:
            state["logits"][:, :, vocab // 3:vocab // 2] = -math.inf
        gaps = torch.rand((groups, beams), generator=gen, device="cuda")
        state["scores"] = -2 - gaps.cumsum(1)
        state["finished"] = torch.rand((groups, beams), generator=gen, device="cuda") < 0.15
        return state
    layers, groups, beams, page = (case[x] for x in ("layers", "groups", "beams", "page"))
    lengths = _lengths(groups, case["low"], case["high"])
    width = -(-case["high"] // page)
    # Each beam has a page of its own for every step of the table, and a spare one.
    pages = groups * beams * (width + 1)
    shape = (layers, pages, case["kv_heads"], page, case["dim"])
    state["k_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    state["v_cache"] = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(groups, beams, width + 1)
    state["tables"], state["spare"] = order[..., :width].contiguous(), order[..., width].contiguous()
    state["parents"] = torch.randint(0, beams, (groups, beams), generator=gen, device="cuda")
    state["parents"][:, 0] = 0
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["host_lengths"] = lengths
    return state


# ----------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _split(state):
    case = state["case"]
    return state["qkv"].split((case["heads"], case["kv_heads"], case["kv_heads"]), 2)


def _own_append(state):
    from exploration_b200 import paged_append
    q, k, v = _split(state)
    rotated = paged_append(q, k, v, state["cos"], state["sin"], state["k_cache"], state["v_cache"],
                           state["tables"], state["positions"])
    return rotated, state["k_cache"], state["v_cache"]


def _own_attention(state):
    from exploration_b200 import paged_attention
    return paged_attention(state["q"], state["k_cache"], state["v_cache"], state["tables"], state["positions"])


def _own_select(state):
    from exploration_b200 import beam_select
    return beam_select(state["logits"], state["scores"], state["finished"], EOS)


def _own_reorder(state):
    from exploration_b200 import beam_reorder
    tables, spare = beam_reorder(state["k_cache"], state["v_cache"], state["tables"], state["spare"],
                                 state["parents"], state["lengths"])
    return state["k_cache"], state["v_cache"], tables, spare


_OWN = {"append": _own_append, "attention": _own_attention, "select": _own_select, "reorder": _own_reorder}


def _rotate(x, cos, sin):
    first, second = x.float().chunk(2, -1)
    return torch.cat((first * cos - second * sin, second * cos + first * sin), -1).to(x.dtype)


def _plain_append(state):
    q, k, v = _split(state)
    positions, page = state["positions"], state["case"]["page"]
    real = positions >= 0
    at = positions.clamp_min(0).long()
    cos, sin = state["cos"][at][:, :, None], state["sin"][at][:, :, None]
    rotated = _rotate(q, cos, sin) * real[:, :, None, None]
    pages = state["tables"].gather(1, at // page).long()
    # Each sequence's new tokens come first in its row.
    for row, count in enumerate(state["counts"]):
        slot = pages[row, :count], slice(None), at[row, :count] % page
        state["k_cache"][slot] = _rotate(k[row, :count], cos[row, :count], sin[row, :count])
        state["v_cache"][slot] = v[row, :count]
    return rotated, state["k_cache"], state["v_cache"]


def _plain_attention(state):
    case, q = state["case"], state["q"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kv
    out = torch.zeros_like(q)
    for row, (n, count) in enumerate(zip(state["lengths"], state["counts"])):
        if count == 0:
            continue
        pages = state["tables"][row, :-(-n // page)].long()
        visible = torch.arange(n, device=q.device) <= state["positions"][row, :count, None]
        step = max(1, kv * 2 ** 31 // (kv * count * group * n))          # key heads at a time
        for lo in range(0, kv, step):
            hi = min(lo + step, kv)
            k = state["k_cache"][pages, lo:hi].transpose(0, 1).reshape(hi - lo, -1, dim)[:, :n].float()
            v = state["v_cache"][pages, lo:hi].transpose(0, 1).reshape(hi - lo, -1, dim)[:, :n].float()
            rows = q[row, :count, lo * group:hi * group].float().view(count, hi - lo, group, dim)
            rows = rows.permute(1, 2, 0, 3).reshape(hi - lo, group * count, dim)
            logits = (rows @ k.transpose(1, 2) / math.sqrt(dim)).view(hi - lo, group, count, n)
            logits = logits.masked_fill_(~visible, -math.inf)
            weights = torch.exp(logits - logits.amax(-1, keepdim=True))
            total = weights.sum(-1, keepdim=True)
            read = (weights.view(hi - lo, group * count, n) @ v).view(hi - lo, group, count, dim) / total
            out[row, :count, lo * group:hi * group] = \
                read.permute(2, 0, 1, 3).reshape(count, (hi - lo) * group, dim).to(q.dtype)
    return out


def _plain_select(state):
    logits, scores, finished = state["logits"].float(), state["scores"], state["finished"]
    groups, beams, vocab = logits.shape
    peak = logits.amax(-1, keepdim=True)
    lse = peak + (logits - peak).exp().sum(-1, keepdim=True).log()
    # The best of each beam, ties to the lowest token, then the best of all, ties to the lowest beam.
    best, token = logits.sort(dim=-1, descending=True, stable=True)
    keep = min(beams, vocab)
    best, token = best[..., :keep], token[..., :keep]
    total = scores[..., None] + (best - lse)
    ended = finished[..., None]
    first = torch.arange(keep, device=logits.device) == 0
    total = torch.where(ended, torch.where(first, scores[..., None], -math.inf), total)
    token = torch.where(ended, EOS, token)
    ranked, order = total.flatten(1).sort(dim=-1, descending=True, stable=True)
    ranked, order = ranked[:, :beams], order[:, :beams]
    parents = order // keep
    tokens = token.flatten(1).gather(1, order)
    return ranked, parents, tokens, finished.gather(1, parents) | (tokens == EOS)


def _plain_reorder(state):
    tables, spare, parents = state["tables"], state["spare"], state["parents"]
    groups, beams, width = tables.shape
    page = state["case"]["page"]
    moved = parents != torch.arange(beams, device=parents.device)
    column = torch.arange(width, device=parents.device)
    tail = (state["lengths"] // page)[:, None]
    taken = tables.gather(1, parents[..., None].expand(-1, -1, width))
    full = column < tail[..., None]
    partial = (state["lengths"] % page != 0)[:, None] & moved
    swap = partial[..., None] & (column == tail[..., None])
    fresh = torch.where(full, taken, torch.where(swap, spare[..., None], tables))
    last = tail.clamp_max(width - 1).expand(-1, beams)[..., None].long()
    freed = torch.where(partial, tables.gather(2, last)[..., 0], spare)
    for group, n in enumerate(state["host_lengths"]):
        rows = n % page
        if rows:
            source = tables[group, parents[group], n // page].long()
            # A beam that stays keeps its page: it is written onto itself.
            target = torch.where(moved[group], spare[group], source).long()
            for cache in (state["k_cache"], state["v_cache"]):
                cache[:, target, :, :rows] = cache[:, source, :, :rows]
    return state["k_cache"], state["v_cache"], fresh, freed


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "select": _plain_select,
          "reorder": _plain_reorder}


# ----------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------

def work(case):
    size = BYTES[case["dtype"]]
    op = case["op"]
    if op == "append":
        tokens = sum(_counts(case))
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        each = 2 * (heads + 2 * kv) * dim * size + 4 * dim + 8     # in and out, one table row, position and page
        padding = (case["batch"] * case["new"] - tokens) * (heads * dim * size + 4)
        return {"bytes": tokens * each + padding, "flops": tokens * 3 * dim * (heads + kv)}
    if op == "attention":
        lengths, counts = _lengths(case["batch"], case["low"], case["high"]), _counts(case)
        keys = sum(n for n, c in zip(lengths, counts) if c)
        pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lengths, counts))
        rows = case["heads"] * case["dim"] * size
        table = sum(-(-n // case["page"]) * 4 for n, c in zip(lengths, counts) if c)
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + sum(counts) * rows
                + case["batch"] * case["new"] * (rows + 4) + table,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if op == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * size + 26), "flops": 3 * rows * case["vocab"]}
    lengths = _lengths(case["groups"], case["low"], case["high"])
    # All but the first beam change their parent for another one in most groups.
    copied = sum((n % case["page"]) * (case["beams"] - 1) for n in lengths)
    kept = 1 - 1 / case["beams"]
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
    beams = case["groups"] * case["beams"]
    return {"bytes": int(2 * copied * kept * row) + beams * (8 * -(-case["high"] // case["page"]) + 16), "flops": 0}


# ----------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return _EXACT[case["op"]](case, state)


def _exact_append(case, state):
    heads, kv, half, page = case["heads"], case["kv_heads"], case["dim"] // 2, case["page"]
    wide = state["qkv"].double()
    k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
    rotated = torch.zeros_like(wide[:, :, :heads])
    for b, count in enumerate(state["counts"]):
        if not count:
            continue
        p = torch.arange(state["lengths"][b] - count, state["lengths"][b], device="cuda")
        # Halves as real and imaginary parts: the rotation is a complex product.
        turn = torch.complex(state["cos"][p].double(), state["sin"][p].double())[:, None]
        x = wide[b, :count, :heads + kv]
        y = torch.view_as_real(torch.complex(x[..., :half], x[..., half:]) * turn)
        y = torch.cat((y[..., 0], y[..., 1]), -1)
        rotated[b, :count] = y[:, :heads]
        where = state["tables"][b].long()[p // page]
        k_cache[where, :, p % page] = y[:, heads:]
        v_cache[where, :, p % page] = wide[b, :count, heads + kv:]
    return rotated, k_cache, v_cache


def _exact_attention(case, state):
    group, page, new = case["heads"] // case["kv_heads"], case["page"], case["new"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, count) in enumerate(zip(state["lengths"], state["counts"])):
        if not count:
            continue
        keys = torch.arange(n, device="cuda")
        place = state["tables"][b].long()[keys // page], keys % page
        for head in range(case["kv_heads"]):
            k = state["k_cache"][place[0], head, place[1]].double()
            v = state["v_cache"][place[0], head, place[1]].double()
            for g in range(head * group, (head + 1) * group):
                a = torch.einsum("rd,nd->rn", state["q"][b, :count, g].double(), k) * case["dim"] ** -0.5
                seen = keys[None] < n - count + 1 + torch.arange(count, device="cuda")[:, None]
                out[b, :count, g] = torch.softmax(a.where(seen, a.new_tensor(-math.inf)), -1) @ v
    return out


def _exact_select(case, state):
    logp = torch.log_softmax(state["logits"].double(), -1)
    total = state["scores"].double()[..., None] + logp
    ended = state["finished"]
    total[ended] = -math.inf
    total[..., EOS] = torch.where(ended, state["scores"].double(), total[..., EOS])
    best = total.flatten(1).topk(case["beams"], -1).values
    return best, None, None, None


def _exact_reorder(case, state):
    k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
    page = case["page"]
    parents, tables, spare = state["parents"].tolist(), state["tables"].tolist(), state["spare"].tolist()
    for g, n in enumerate(state["host_lengths"]):
        for beam, parent in enumerate(parents[g]):
            if parent != beam and n % page:
                source, target = tables[g][parent][n // page], spare[g][beam]
                for cache in (k_cache, v_cache):
                    cache[:, target, :, :n % page] = cache[:, source, :, :n % page]
    return k_cache, v_cache, None, None


_EXACT = {"append": _exact_append, "attention": _exact_attention, "select": _exact_select,
          "reorder": _exact_reorder}
