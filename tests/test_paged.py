"""Paged-cache and beam operators on the CPU: definitions against plain loops, and refusals."""
import math

import pytest
import torch

import exploration_b200 as eb


def small_cache(lengths, kv=2, dim=8, page=16, dtype=torch.float64, seed=0):
    gen = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(needed), generator=gen).to(torch.int32)
    k = torch.randn(sum(needed), kv, page, dim, generator=gen, dtype=dtype)
    v = torch.randn(sum(needed), kv, page, dim, generator=gen, dtype=dtype)
    tables = torch.full((len(lengths), max(needed)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(needed):
        tables[b, :n] = order[at:at + n]
        at += n
    return k, v, tables


def test_attention_against_a_loop_over_rows_and_keys():
    lengths, page, group, dim = [20, 1, 33], 16, 3, 8
    k, v, tables = small_cache(lengths)
    q = torch.randn(3, 4, 2 * group, dim, dtype=torch.float64)
    positions = torch.tensor([[19, 0, 16, 15], [0, -1, -1, -1], [-1, 32, -1, 7]], dtype=torch.int32)
    out = eb.paged_attention(q, k, v, tables, positions)
    for b in range(3):
        for t in range(4):
            for h in range(2 * group):
                p = int(positions[b, t])
                if p < 0:
                    assert not out[b, t, h].any()
                    continue
                weights, values = [], []
                for i in range(p + 1):
                    place = int(tables[b, i // page]), h // group, i % page
                    weights.append(math.exp(float(q[b, t, h] @ k[place]) / math.sqrt(dim)))
                    values.append(v[place])
                want = sum(w * x for w, x in zip(weights, values)) / sum(weights)
                torch.testing.assert_close(out[b, t, h], want, atol=1e-12, rtol=1e-12)


def test_append_rotates_like_the_models_embedding_and_fills_pages():
    from exploration_b200.models.blocks import RotaryEmbedding
    rope = RotaryEmbedding(8)
    k_cache, v_cache, tables = small_cache([40, 20], dtype=torch.float32)
    qkv = torch.randn(2, 5, 8, 8)
    q, k, v = qkv.split((4, 2, 2), 2)
    positions = torch.tensor([[14, 15, 16, 17, 18], [3, -1, -1, -1, -1]])
    cos, sin = rope.tables(torch.arange(64))
    before = k_cache.clone()
    out = eb.paged_append(q, k, v, cos, sin, k_cache, v_cache, tables, positions)
    torch.testing.assert_close(out[0], rope(q[0], positions[0]))
    turned = rope(k[0], positions[0])
    for i, p in enumerate(positions[0].tolist()):
        page = int(tables[0, p // 16])
        torch.testing.assert_close(k_cache[page, :, p % 16], turned[i])
        assert torch.equal(v_cache[page, :, p % 16], v[0, i])
    assert not out[1, 1:].any()
    changed = (k_cache != before).any(-1).any(1).sum()
    assert int(changed) == 6


def test_append_then_attention_equals_causal_attention():
    """A prompt taken in chunks of any size gives the whole prompt's causal attention."""
    from exploration_b200.models.blocks import RotaryEmbedding
    rope, n = RotaryEmbedding(8), 37
    k_cache, v_cache, tables = small_cache([n])
    cos, sin = rope.tables(torch.arange(n))
    q, k, v = torch.randn(1, n, 6, 8, dtype=torch.float64).split(2, 2)
    parts = []
    for lo, hi in ((0, 1), (1, 18), (18, 36), (36, 37)):
        positions = torch.arange(lo, hi, dtype=torch.int32)[None]
        turned = eb.paged_append(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], cos, sin, k_cache, v_cache, tables, positions)
        parts.append(eb.paged_attention(turned, k_cache, v_cache, tables, positions))
    at = torch.arange(n)
    angle = [t.double() for t in (cos, sin)]
    from exploration_b200.ops.paged import rotate_reference as rotate
    want = torch.nn.functional.scaled_dot_product_attention(
        *(rotate(t, angle[0][at], angle[1][at]).transpose(1, 2) for t in (q, k)), v.transpose(1, 2),
        is_causal=True).transpose(1, 2)
    torch.testing.assert_close(torch.cat(parts, 1), want, atol=1e-6, rtol=1e-6)


def test_select_against_all_candidates():
    torch.manual_seed(0)
    logits, scores = torch.randn(5, 3, 11, dtype=torch.float64), -torch.rand(5, 3)
    finished = torch.zeros(5, 3, dtype=torch.bool)
    finished[1, 0] = finished[2, 2] = True
    got, parents, tokens, ended = eb.beam_select(logits, scores, finished, 4)
    for g in range(5):
        pool = []
        for w in range(3):
            if finished[g, w]:
                pool.append((-float(scores[g, w]), w, 4))
                continue
            logp = torch.log_softmax(logits[g, w], -1)
            pool += [(-(float(scores[g, w]) + float(logp[t])), w, t) for t in range(11)]
        for i, (total, w, t) in enumerate(sorted(pool)[:3]):
            assert (int(parents[g, i]), int(tokens[g, i])) == (w, t)
            assert abs(float(got[g, i]) + total) < 1e-6
            assert bool(ended[g, i]) == (bool(finished[g, w]) or t == 4)


def test_select_more_beams_than_tokens():
    got, parents, tokens, _ = eb.beam_select(torch.zeros(1, 3, 2), torch.tensor([[0.0, -math.inf, -math.inf]]),
                                             torch.zeros(1, 3, dtype=torch.bool), -1)
    assert tokens[0, :2].tolist() == [0, 1] and parents[0].tolist() == [0, 0, 1]
    assert math.isinf(got[0, 2])


def test_reorder_moves_states_and_keeps_shared_pages():
    page = 16
    k = torch.arange(2 * 12 * 1 * page * 2, dtype=torch.float32).view(2, 12, 1, page, 2)
    v = -k
    tables = torch.arange(9, dtype=torch.int32).view(1, 3, 3)
    spare = torch.arange(9, 12, dtype=torch.int32).view(1, 3)
    parents = torch.tensor([[1, 1, 0]])
    before = k.clone()
    fresh, freed = eb.beam_reorder(k, v, tables, spare, parents, torch.tensor([21], dtype=torch.int32))
    assert fresh.tolist() == [[[3, 9, 2], [3, 4, 5], [0, 11, 8]]]
    assert freed.tolist() == [[1, 10, 7]]
    assert torch.equal(k[:, 9, :, :5], before[:, 4, :, :5]) and torch.equal(k[:, 11, :, :5], before[:, 1, :, :5])
    assert torch.equal(k[:, 9, :, 5:], before[:, 9, :, 5:]) and torch.equal(v, -k)
    assert torch.equal(k[:, :9], before[:, :9])


def refuse(message, call, *args):
    with pytest.raises(ValueError, match=message):
        call(*args)


def test_paged_refusals():
    k, v, tables = small_cache([20], dtype=torch.float32)
    q, positions = torch.randn(1, 2, 4, 8), torch.zeros(1, 2, dtype=torch.int32)
    good = [q, k, v, tables, positions]

    def with_(**changes):
        names = ["q", "k", "v", "tables", "positions"]
        return [changes.get(n, x) for n, x in zip(names, good)]

    eb.paged_attention(*good)
    attend = eb.paged_attention
    refuse("expected rows", attend, *with_(q=q[0]))
    refuse("expected rows", attend, *with_(v=v[:, :1]))
    refuse("expected rows", attend, *with_(q=q[..., :6]))
    refuse("power of two", attend, *with_(k=k[:, :, :8], v=v[:, :, :8]))
    refuse("power of two", attend, *with_(k=torch.zeros(2, 2, 24, 8), v=torch.zeros(2, 2, 24, 8)))
    refuse("head_dim", attend, torch.zeros(1, 2, 4, 7), torch.zeros(2, 2, 16, 7), torch.zeros(2, 2, 16, 7), tables,
           positions)
    refuse("head_dim", attend, torch.zeros(1, 2, 4, 258), torch.zeros(2, 2, 16, 258), torch.zeros(2, 2, 16, 258),
           tables, positions)
    refuse("multiple", attend, *with_(q=torch.zeros(1, 2, 3, 8)))
    refuse("positions", attend, *with_(positions=positions[:, :1]))
    refuse("positions", attend, *with_(tables=tables[0]))
    refuse("int32", attend, *with_(positions=positions.float()))
    refuse("int32", attend, *with_(tables=tables.long()))
    refuse("one dtype", attend, *with_(q=q.double()))
    refuse("no gradient", attend, *with_(q=q.clone().requires_grad_()))
    refuse("one device", attend, *with_(tables=tables.to("meta")))
    cos = torch.zeros(20, 4)
    new = torch.randn(1, 2, 2, 8)
    append = eb.paged_append
    append(q, new, new, cos, cos, k, v, tables, positions)
    refuse("k, v", append, q, new[:, :1], new[:, :1], cos, cos, k, v, tables, positions)
    refuse("match in dtype", append, q, new.double(), new.double(), cos, cos, k, v, tables, positions)
    refuse("cos, sin", append, q, new, new, cos[:, :3], cos[:, :3], k, v, tables, positions)
    refuse("cos, sin", append, q, new, new, cos.double(), cos.double(), k, v, tables, positions)
    refuse("no gradient", append, q, new, new.clone().requires_grad_(), cos, cos, k, v, tables, positions)


def test_beam_refusals():
    logits, scores, ended = torch.zeros(2, 3, 5), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)
    refuse("expected logits", eb.beam_select, logits[0], scores, ended, 0)
    refuse("expected logits", eb.beam_select, logits, scores[:, :2], ended, 0)
    refuse("fp32", eb.beam_select, logits, scores.double(), ended, 0)
    refuse("bool", eb.beam_select, logits, scores, ended.int(), 0)
    refuse("eos", eb.beam_select, logits, scores, ended, 5)
    refuse("eos", eb.beam_select, logits, scores, ended, -2)
    refuse("beams", eb.beam_select, torch.zeros(1, 33, 5), torch.zeros(1, 33), torch.zeros(1, 33, dtype=torch.bool), 0)
    refuse("no gradient", eb.beam_select, logits.clone().requires_grad_(), scores, ended, 0)
    pool = torch.zeros(1, 8, 1, 16, 2)
    tables, spare = torch.zeros(2, 3, 1, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    parents, lengths = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    refuse("expected pools", eb.beam_reorder, pool[0], pool[0], tables, spare, parents, lengths)
    refuse("expected pools", eb.beam_reorder, pool, pool, tables, spare[:1], parents, lengths)
    refuse("int64", eb.beam_reorder, pool, pool, tables, spare, parents.int(), lengths)
    refuse("contiguous", eb.beam_reorder, pool.transpose(3, 4), pool.transpose(3, 4), tables, spare, parents, lengths)
    refuse("one dtype", eb.beam_reorder, pool, pool.double(), tables, spare, parents, lengths)
