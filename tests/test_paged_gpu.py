"""Paged-cache and beam kernels against their definitions in 64 bits (B200 only)."""
import math

import pytest
import torch

from exploration_b200.ops import beam, paged

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# Unit roundoffs of the output type and of a probability on its way into the second product.
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _clean_errors(native):
    yield
    assert native.device_errors(torch.cuda.current_device()) == (0, 0)


def make_cache(lengths, kv, dim, page, dtype, seed=0, garbage=math.nan, width=None, extra=3):
    """Pools whose written rows are N(0, 1) and all others ``garbage``; unused table entries are invalid."""
    gen = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lengths]
    pages = sum(needed) + extra
    order = torch.randperm(pages, generator=gen)
    k = torch.full((pages, kv, page, dim), garbage, dtype=torch.float64)
    v = k.clone()
    tables = torch.full((len(lengths), width or max(1, max(needed))), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        ids = order[at:at + needed[b]]
        at += needed[b]
        tables[b, :needed[b]] = ids.to(torch.int32)
        for j, i in enumerate(ids.tolist()):
            rows = min(page, n - j * page)
            k[i, :, :rows] = torch.randn(kv, rows, dim, generator=gen, dtype=torch.float64)
            v[i, :, :rows] = torch.randn(kv, rows, dim, generator=gen, dtype=torch.float64)
    return k.to(dtype).cuda(), v.to(dtype).cuda(), tables.cuda()


def check_attention(q, k, v, tables, positions):
    out = paged.paged_attention(q, k, v, tables, positions)
    assert out.shape == q.shape and out.dtype == q.dtype
    host = [t.double().cpu() if t.is_floating_point() else t.cpu() for t in (q, k, v, tables, positions)]
    want = paged.attention_reference(*host)
    # Mean of |v| under the row's weights: every error of a weight is bounded relative to it.
    mass = paged.attention_reference(host[0], host[1], host[2].abs(), *host[3:])
    u = ROUND[q.dtype]
    # Weights rounded to the input type, the result rounded once; 4e-5: fp32 logits of size about 30
    # (each off by at most head_dim * 2^-24 of the sum of its terms' sizes) and the hardware exponential.
    bound = u * want.abs() + ((u if q.dtype != torch.float32 else 0.0) + 4e-5) * mass + 1e-30
    error = (out.double().cpu() - want).abs()
    assert bool((error <= bound).all()), float((error / bound).max())
    return out


def queries(batch, new, heads, dim, dtype, seed=1, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(batch, new, heads, dim, generator=gen)).to(dtype).cuda()


def tail_positions(lengths, counts, new):
    rows = torch.full((len(lengths), new), -1, dtype=torch.int32)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        rows[b, :c] = torch.arange(n - c, n)
    return rows.cuda()


# lengths, new tokens (each sequence's count below), heads, kv_heads, dim, page
CASES = [
    ([1], [1], 1, 4, 4, 64, 16),
    ([2, 17, 300, 64, 65], [1] * 5, 1, 4, 4, 64, 16),
    ([1000, 3, 2049], [1] * 3, 1, 8, 2, 128, 64),
    ([129, 640], [1, 1], 1, 6, 2, 64, 32),
    ([500, 77, 16], [5, 0, 3], 5, 4, 4, 64, 16),
    ([333, 90], [4, 4], 4, 16, 4, 128, 128),
    ([40, 41], [16, 9], 16, 2, 2, 64, 256),
    ([17, 530], [17, 20], 20, 4, 2, 64, 16),
    ([129, 600, 300], [129, 100, 0], 130, 4, 4, 64, 32),
    ([700, 1500], [300, 257], 300, 8, 2, 128, 64),
    ([257], [257], 257, 12, 4, 64, 64),
    ([900], [33], 33, 20, 4, 128, 16),
    ([300, 20], [7, 20], 20, 34, 2, 64, 32),
    ([70, 5], [3, 2], 3, 2, 1, 16, 16),
    ([70, 200], [1, 1], 1, 3, 1, 256, 32),
    ([65, 130], [40, 40], 40, 2, 2, 96, 64),
    ([33], [5], 5, 2, 2, 6, 16),
    ([33, 90], [2, 1], 2, 2, 2, 32, 16),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,counts,new,heads,kv,dim,page", CASES)
def test_attention_matches_definition(lengths, counts, new, heads, kv, dim, page, dtype):
    k, v, tables = make_cache(lengths, kv, dim, page, dtype)
    out = check_attention(queries(len(lengths), new, heads, dim, dtype), k, v, tables,
                          tail_positions(lengths, counts, new))
    for b, count in enumerate(counts):
        assert not out[b, count:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,heads,kv", [(1, 4, 4), (3, 8, 2), (40, 4, 2), (150, 4, 4)])
def test_attention_any_positions(new, heads, kv, dtype):
    """Rows in any order, padding anywhere, a sequence without rows, a table wider than needed."""
    lengths = [200, 75, 1, 130]
    k, v, tables = make_cache(lengths, kv, 64, 32, dtype, seed=5, width=11)
    gen = torch.Generator().manual_seed(3)
    positions = torch.stack([torch.randint(-1, n, (new,), generator=gen) for n in lengths]).to(torch.int32)
    positions[:, 0] = torch.tensor([199, 74, 0, -1])
    positions[3] = -1
    out = check_attention(queries(4, new, heads, 64, dtype), k, v, tables, positions.cuda())
    assert not out[3].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 6, 64])
def test_attention_extreme_logits(new, dtype):
    """One key far above all others, and rows whose logits are all far below zero."""
    lengths = [350, 200]
    k, v, tables = make_cache(lengths, 2, 64, 16, dtype, seed=9)
    q = queries(2, new, 4, 64, dtype)
    page = int(tables[0, 3])
    k[page, :, 5] = q[0, -1, ::2] * 4       # about 4 * 4 * 64 / 8 = 128 above the rest for one row
    positions = tail_positions(lengths, [new, new], new)
    out = check_attention(q, k, v, tables, positions)
    torch.testing.assert_close(out[0, -1, 0].float(), v[page, 0, 5].float(), atol=1e-3, rtol=1e-2)
    # softmax does not change when all logits of a row move together
    k2 = k.clone()
    k2[:, :, :, 0] = torch.where(k2[:, :, :, 0].isnan(), k2[:, :, :, 0], torch.full_like(k2[:, :, :, 0], 64.0))
    q2 = q.clone()
    q2[..., 0] = -64.0                       # -512 on every logit
    check_attention(q2, k2, v, tables, positions)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_off_the_vector_grid(new, dtype):
    """Queries and pools that start between 16-byte boundaries, and strided queries."""
    lengths = [90, 300]
    k, v, tables = make_cache(lengths, 2, 64, 16, dtype)
    q, positions = queries(2, new, 4, 64, dtype), tail_positions(lengths, [new, new], new)

    def shifted(t):
        base = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        base[1:] = t.flatten()
        return base[1:].view(t.shape)

    check_attention(shifted(q), k, v, tables, positions)
    check_attention(q, shifted(k), shifted(v), tables, positions)
    wide = torch.cat((q, q), 2)[:, :, 4:]
    assert not wide.is_contiguous()
    check_attention(wide, k, v, tables, positions)


def test_attention_split_is_deterministic_and_streams():
    lengths = [5000, 20, 3000]
    k, v, tables = make_cache(lengths, 4, 64, 64, torch.bfloat16)
    q, positions = queries(3, 1, 8, 64, torch.bfloat16), tail_positions(lengths, [1] * 3, 1)
    first = check_attention(q, k, v, tables, positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [paged.paged_attention(q, k, v, tables, positions) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(first, x) for x in again)


def test_attention_graph_follows_positions():
    """A captured step serves later steps: only device data says how long a sequence is."""
    lengths = [700, 45]
    k, v, tables = make_cache(lengths, 2, 128, 32, torch.bfloat16)
    q = queries(2, 1, 4, 128, torch.bfloat16)
    positions = tail_positions([12, 3], [1, 1], 1)
    paged.paged_attention(q, k, v, tables, positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.paged_attention(q, k, v, tables, positions)
    for step in ([12, 3], [699, 44], [0, -1], [64, 31]):
        positions.copy_(torch.tensor(step, dtype=torch.int32)[:, None])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged.paged_attention(q, k, v, tables, positions))


def test_attention_many_sequences():
    """More sequences than the split's table holds."""
    lengths = [1 + (i * 37) % 90 for i in range(2100)]
    k, v, tables = make_cache(lengths, 1, 64, 16, torch.bfloat16)
    q = queries(2100, 1, 2, 64, torch.bfloat16)
    positions = tail_positions(lengths, [1] * 2100, 1)
    positions[7] = -1
    out = check_attention(q, k, v, tables, positions)
    assert not out[7].any()


def test_attention_pool_past_32_bits():
    """Pages whose element offsets pass 2^31 (a 4.6 GB pool per tensor)."""
    pages, kv, page, dim = 18000, 8, 128, 128
    k = torch.zeros(pages, kv, page, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    ids = torch.tensor([[17999, 16500, 3]], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    k[ids[0].long()] = torch.randn(3, kv, page, dim, generator=gen, device="cuda").to(k.dtype)
    v[ids[0].long()] = torch.randn(3, kv, page, dim, generator=gen, device="cuda").to(k.dtype)
    small_k, small_v = k[ids[0].long()].contiguous(), v[ids[0].long()].contiguous()
    small = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    for new in (1, 40):
        q, positions = queries(1, new, 8, dim, torch.bfloat16), tail_positions([300], [new], new)
        assert torch.equal(paged.paged_attention(q, k, v, ids, positions),
                           paged.paged_attention(q, small_k, small_v, small, positions))
    half = dim // 2
    cos, sin = torch.ones(512, half, device="cuda"), torch.zeros(512, half, device="cuda")
    rows = torch.randn(1, 1, kv, dim, device="cuda", generator=gen).to(k.dtype)
    position = torch.tensor([[130]], dtype=torch.int32, device="cuda")
    paged.paged_append(rows, rows, rows, cos, sin, k, v, ids, position)
    assert torch.equal(k[16500, :, 2], rows[0, 0]) and torch.equal(v[16500, :, 2], rows[0, 0])


# ----------------------------------------------------------------------------
# append
# ----------------------------------------------------------------------------

APPEND = [
    (1, 1, 4, 4, 64, 16, False), (3, 7, 8, 2, 128, 32, True), (2, 33, 6, 2, 64, 64, True),
    (2, 5, 3, 1, 96, 16, False), (2, 4, 2, 2, 6, 16, True), (1, 3, 2, 1, 16, 16, True), (2, 70, 2, 2, 256, 128, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,new,heads,kv,dim,page,strided", APPEND)
def test_append_matches_definition(batch, new, heads, kv, dim, page, strided, dtype):
    gen = torch.Generator().manual_seed(4)
    lengths = [new + 11 * (b + 1) for b in range(batch)]
    k_cache, v_cache, tables = make_cache(lengths, kv, dim, page, dtype, garbage=0.5)
    qkv = torch.randn(batch, new, heads + 2 * kv, dim, generator=gen).to(dtype).cuda()
    q, k, v = qkv.split((heads, kv, kv), 2)
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    positions = tail_positions(lengths, [max(0, new - 2 * b) for b in range(batch)], new)
    angle = torch.arange(max(lengths))[:, None] * 10_000.0 ** (-torch.arange(0, dim, 2) / dim)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    host = [t.double().cpu() for t in (q, k, v, cos, sin, k_cache, v_cache)]
    want = paged.append_reference(*host, tables.cpu(), positions.cpu())
    got = paged.paged_append(q, k, v, cos, sin, k_cache, v_cache, tables, positions)
    # Two fp32 products and one sum of terms of size at most |x1| + |x2| (3 roundings), then one rounding.
    size = qkv.abs().max().double().cpu() * 2
    for mine, exact in ((got, want), (k_cache, host[5])):
        bound = ROUND[dtype] * exact.abs() + 3 * 2.0 ** -24 * size
        assert bool(((mine.double().cpu() - exact).abs() <= bound).all())
    assert torch.equal(v_cache.double().cpu(), host[6])


def test_append_misaligned_views_and_bad_rows():
    """Views off the 16-byte grid; rows outside the tables leave the cache alone."""
    dtype, page = torch.bfloat16, 16
    k_cache, v_cache, tables = make_cache([40], 2, 64, page, dtype, garbage=0.25)
    base = torch.randn(1 * 3 * 4 * 64 + 3, device="cuda").to(dtype)
    q = base[3:].view(1, 3, 4, 64)
    k, v = q[:, :, :2], q[:, :, 2:]
    cos, sin = torch.rand(48, 32, device="cuda"), torch.rand(48, 32, device="cuda")
    positions = torch.tensor([[39, 1000, -1]], dtype=torch.int64, device="cuda")
    before = k_cache.clone()
    out = paged.paged_append(q, k, v, cos, sin, k_cache, v_cache, tables, positions)
    ref_k, ref_v = before.cpu(), v_cache.cpu()
    want = paged.append_reference(*(t.cpu() for t in (q[:, :1], k[:, :1], v[:, :1], cos, sin)), ref_k, ref_v,
                                  tables.cpu(), positions[:, :1].cpu())
    torch.testing.assert_close(out[:, :1].cpu(), want, atol=0, rtol=2.0 ** -7)
    assert not out[:, 1:].any()
    torch.testing.assert_close(k_cache.cpu(), ref_k, atol=0, rtol=2.0 ** -7)
    assert torch.equal(v_cache.cpu(), ref_v)


# ----------------------------------------------------------------------------
# beams
# ----------------------------------------------------------------------------

def select_inputs(groups, beams, vocab, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    logits = (3 * torch.randn(groups, beams, vocab, generator=gen)).to(dtype)
    scores = -2 - torch.rand(groups, beams, generator=gen).cumsum(1)
    finished = torch.rand(groups, beams, generator=gen) < 0.2
    return logits, scores, finished


def check_select(logits, scores, finished, eos):
    got = beam.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), eos)
    want = beam.select_reference(logits.double(), scores, finished, eos)
    # lse: 3 ulp of a sum of fp32 exponentials (4e-7), then two roundings of numbers below 2^6.
    torch.testing.assert_close(got[0].cpu(), want[0].float(), atol=2e-5, rtol=0)
    for mine, exact in zip(got[1:], want[1:]):
        assert torch.equal(mine.cpu(), exact)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,beams,vocab", [
    (1, 1, 1), (2, 4, 2), (3, 4, 256), (1, 8, 1000), (2, 5, 1017), (2, 3, 1024), (2, 3, 1025), (2, 2, 8191),
    (3, 8, 8193), (2, 32, 20011), (1, 3, 100003), (2, 31, 40)])
def test_select_matches_definition(groups, beams, vocab, dtype):
    check_select(*select_inputs(groups, beams, vocab, dtype, seed=vocab), eos=0 if vocab < 3 else 2)


@pytest.mark.parametrize("vocab", [40, 9000])
def test_select_ties_go_to_the_lowest(vocab):
    logits = torch.zeros(2, 3, vocab)
    logits[1, :, 5::7] = 1.0
    logits[1, :, 0] = -0.0
    scores = torch.full((2, 3), -1.0)
    finished = torch.zeros(2, 3, dtype=torch.bool)
    got = beam.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), -1)
    assert got[1].tolist() == [[0, 0, 0], [0, 0, 0]]
    assert got[2].tolist() == [[0, 1, 2], [5, 12, 19]]
    assert not got[3].any()


@pytest.mark.parametrize("vocab", [50, 9000])
def test_select_masked_and_dead_beams(vocab):
    """Masked tokens are never preferred; beams without a finite sum offer nothing; ended beams stay."""
    logits, scores, _ = select_inputs(4, 4, vocab, torch.float32)
    finished = torch.zeros(4, 4, dtype=torch.bool)
    logits[0, 0] = -math.inf                     # nothing left
    logits[0, 1, 3] = math.nan
    logits[0, 2, 3] = math.inf
    logits[1, :, 7:] = -math.inf
    logits[1, :, 2] = torch.finfo(torch.float32).min
    finished[2] = True                           # all ended
    finished[3, 0] = True
    scores[3, 1] = -math.inf                     # a beam that does not exist yet
    check_select(logits, scores, finished, eos=4)


@pytest.mark.parametrize("vocab", [50, 9000])
def test_select_all_beams_dead(vocab):
    logits = torch.full((2, 3, vocab), -math.inf)
    logits[1, :, 4] = math.nan
    check_select(logits, torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool), eos=1)


@pytest.mark.parametrize("vocab", [900, 30000])
def test_select_best_tokens_side_by_side(vocab):
    """Many of the best logits in few lanes, in rising, falling and equal runs."""
    logits = torch.randn(3, 8, vocab, generator=torch.Generator().manual_seed(2))
    logits[0, :, 100:300] = torch.linspace(9, 12, 200)
    logits[1, :, 100:300] = torch.linspace(12, 9, 200)
    logits[2, :, 64:320] = 10.0
    check_select(logits, -torch.rand(3, 8).cumsum(1), torch.zeros(3, 8, dtype=torch.bool), eos=-1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,groups,beams,kv,dim,page,lengths", [
    (1, 1, 1, 1, 64, 16, [5]), (2, 3, 4, 2, 64, 16, [1, 16, 31]), (3, 2, 6, 4, 64, 32, [63, 64]),
    (2, 2, 3, 3, 6, 16, [20, 0]), (1, 1, 32, 1, 128, 16, [17])])
def test_reorder_matches_definition(layers, groups, beams, kv, dim, page, lengths, dtype):
    gen = torch.Generator().manual_seed(8)
    width = max(1, -(-max(lengths) // page))
    pages = groups * beams * (width + 1)
    k = torch.randn(layers, pages, kv, page, dim, generator=gen).to(dtype)
    v = torch.randn(layers, pages, kv, page, dim, generator=gen).to(dtype)
    order = torch.randperm(pages, generator=gen).to(torch.int32).view(groups, beams, width + 1)
    tables, spare = order[..., :width].contiguous(), order[..., width].contiguous()
    parents = torch.randint(0, beams, (groups, beams), generator=gen)
    n = torch.tensor(lengths, dtype=torch.int32)
    device = [t.cuda() for t in (k, v, tables, spare, parents, n)]
    got = beam.beam_reorder(*device)
    want = beam.reorder_reference(k, v, tables, spare, parents, n)
    for mine, exact in zip((device[0], device[1], *got), (k, v, *want)):
        assert torch.equal(mine.cpu(), exact)
    assert torch.equal(device[2].cpu(), tables) and torch.equal(device[3].cpu(), spare)


# ----------------------------------------------------------------------------
# refusals
# ----------------------------------------------------------------------------

def test_native_refusals_are_the_same():
    k, v, tables = make_cache([20], 2, 8, 16, torch.float32)
    q, positions = torch.randn(1, 2, 4, 8, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    new, cos = torch.randn(1, 2, 2, 8, device="cuda"), torch.zeros(20, 4, device="cuda")

    def refuse(message, call, *args):
        with pytest.raises(ValueError, match=message):
            call(*args)

    attend, append = paged.paged_attention, paged.paged_append
    refuse("expected rows", attend, q[0], k, v, tables, positions)
    refuse("expected rows", attend, q, k, v[:, :1], tables, positions)
    refuse("power of two", attend, q, k[:, :, :8], v[:, :, :8], tables, positions)
    refuse("head_dim", attend, q[..., :7], k[..., :7], v[..., :7], tables, positions)
    refuse("multiple", attend, q[:, :, :3], k, v, tables, positions)
    refuse("positions", attend, q, k, v, tables, positions[:, :1])
    refuse("int32", attend, q, k, v, tables.long(), positions)
    refuse("one dtype", attend, q.half(), k, v, tables, positions)
    refuse("one device", attend, q, k, v, tables.cpu(), positions)
    refuse("no gradient", attend, q.clone().requires_grad_(), k, v, tables, positions)
    refuse("fp32, fp16 or bf16", attend, q.double(), k.double(), v.double(), tables, positions)
    refuse("contiguous", attend, q, k.transpose(0, 1).contiguous().transpose(0, 1), v, tables, positions)
    refuse("k, v", append, q, new[:, :1], new[:, :1], cos, cos, k, v, tables, positions)
    refuse("match in dtype", append, q, new.half(), new.half(), cos, cos, k, v, tables, positions)
    refuse("cos, sin", append, q, new, new, cos.double(), cos.double(), k, v, tables, positions)
    logits, scores = torch.zeros(2, 3, 5, device="cuda"), torch.zeros(2, 3, device="cuda")
    ended = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    refuse("expected logits", beam.beam_select, logits[0], scores, ended, 0)
    refuse("fp32", beam.beam_select, logits, scores.half(), ended, 0)
    refuse("eos", beam.beam_select, logits, scores, ended, 5)
    refuse("beams", beam.beam_select, torch.zeros(1, 33, 5, device="cuda"), torch.zeros(1, 33, device="cuda"),
           torch.zeros(1, 33, dtype=torch.bool, device="cuda"), 0)
    refuse("no gradient", beam.beam_select, logits.clone().requires_grad_(), scores, ended, 0)
    pool = torch.zeros(1, 8, 1, 16, 2, device="cuda")
    table, spare = torch.zeros(2, 3, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, dtype=torch.int32,
                                                                                       device="cuda")
    parents, lengths = spare.long(), torch.zeros(2, dtype=torch.int32, device="cuda")
    refuse("expected pools", beam.beam_reorder, pool[0], pool[0], table, spare, parents, lengths)
    refuse("int64", beam.beam_reorder, pool, pool, table, spare, parents.int(), lengths)
    refuse("contiguous", beam.beam_reorder, pool.transpose(3, 4), pool.transpose(3, 4), table, spare, parents, lengths)


def test_empty_calls():
    k, v, tables = make_cache([20], 2, 64, 16, torch.bfloat16)
    none = torch.zeros(1, 0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert paged.paged_attention(none, k, v, tables, torch.zeros(1, 0, dtype=torch.int32, device="cuda")).numel() == 0
    q = torch.ones(1, 2, 4, 64, device="cuda", dtype=torch.bfloat16)
    hidden = torch.full((1, 2), -1, dtype=torch.int32, device="cuda")
    assert not paged.paged_attention(q, k, v, tables, hidden).any()
    assert not paged.paged_attention(q, k[:0], v[:0], tables, hidden).any()
    assert not paged.paged_attention(q, k, v, tables[:, :0], hidden).any()
