"""Decoding kernels at their edges, against their definitions in 64 bits (B200 only)."""
import pytest
import torch

import exploration_b200 as eb
from tests.test_decoding_edges import (EMPTY_POOLS, REORDERED, check_gradients_are_refused, lowest_masked,
                                       reorder_inputs)
from tests.test_paged_gpu import check_attention, check_select, make_cache, queries, select_inputs, tail_positions

pytestmark = pytest.mark.gpu
SIXTEEN = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _clean_errors(native):
    yield
    assert native.device_errors(torch.cuda.current_device()) == (0, 0)


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,heads,kv", [(20, 2, 2), (128, 2, 1), (300, 2, 2)])
def test_attention_items_of_few_tiles(new, heads, kv, dim, dtype):
    """Chunks over one to five key tiles, rows for one and for both softmax warpgroups, many items a CTA."""
    lengths = [1, 100, 128, 129, 256, 257, 300, 384, 385, 512, 513, 640] * 8
    k, v, tables = make_cache(lengths, kv, dim, 16, dtype, seed=3)
    positions = tail_positions(lengths, [min(n, new) for n in lengths], new)
    q = queries(len(lengths), new, heads, dim, dtype)
    out = check_attention(q, k, v, tables, positions)
    for _ in range(20):
        assert torch.equal(out, eb.paged_attention(q, k, v, tables, positions))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab,spans", [
    (50, [(5, 20)]), (50, [(0, 49)]), (1000, [(0, 1000)]), (1024, [(1, 1023)]),
    (9000, [(3000, 5200)]), (9000, [(8192, 9000)]), (9000, [(0, 8192)]), (9000, [(2, 9000)]),
    (20011, [(0, 16384)]), (20011, [(1, 20010)]), (30000, [(8000, 30000)])])
def test_select_with_the_types_lowest_value_as_a_mask(vocab, spans, dtype):
    """Spans, chunks and whole rows at the lowest finite value weigh nothing beside others, and are no dead beams."""
    scores, ended = -torch.rand(2, 3).cumsum(1), torch.zeros(2, 3, dtype=torch.bool)
    check_select(lowest_masked(dtype, vocab, spans), scores, ended, eos=-1)
    check_select(lowest_masked(dtype, vocab, spans).neg(), scores, ended, eos=-1)


@pytest.mark.parametrize("vocab", [300, 9000])
def test_select_logits_far_from_zero(vocab):
    """The log-probability is taken from the distance to the largest logit: no bits are lost to its size."""
    logits = torch.randn(2, 3, vocab, generator=torch.Generator().manual_seed(1)) + 2.0 ** 16
    check_select(logits, -torch.rand(2, 3).cumsum(1), torch.zeros(2, 3, dtype=torch.bool), eos=-1)


def test_select_many_beams_over_a_large_vocabulary():
    """More chunk entries than the joining warp holds (32 beams x 13 chunks)."""
    for beams in (20, 32):
        check_select(*select_inputs(2, beams, 100003, torch.bfloat16, seed=beams), eos=2)
    logits, scores, ended = select_inputs(1, 32, 100003, torch.float32)
    logits[0, 3] = 1.5                       # ties over all chunks
    logits[0, 4, 40:] = -float("inf")
    check_select(logits, scores, ended, eos=2)


@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("gap", [4, 10, 14, 17, 19])
@pytest.mark.parametrize("sink", [0, 700, 1499])
@pytest.mark.parametrize("new,heads", [(1, 2), (5, 4), (40, 2), (300, 2)])
def test_attention_one_key_takes_nearly_all_weight(new, heads, sink, gap, dim, dtype):
    """A key of value zero ``gap`` (natural logarithm) above all others: the result is what the others hold."""
    lengths = [1500 + new, 1800]
    k, v, tables = make_cache(lengths, 2, dim, 64, dtype, seed=4)
    k.mul_(0.05)
    v.copy_(64 + 16 * v)                      # of one sign: a loss common to all weights does not average out
    q = queries(2, new, heads, dim, dtype, scale=0.05)
    q[..., 0] = 4.0
    for b in range(2):
        page, row = int(tables[b, sink // 64]), sink % 64
        k[page, :, row] = 0
        k[page, :, row, 0] = gap * dim ** 0.5 / 4
        v[page, :, row] = 0
    check_attention(q, k, v, tables, tail_positions(lengths, [new, new], new))


@pytest.mark.parametrize("shape", EMPTY_POOLS + [(2, 12, 2, 16, 8)])
def test_reorder_of_empty_pools(shape):
    fresh, freed = eb.beam_reorder(*reorder_inputs(shape, "cuda"))
    assert (fresh.tolist(), freed.tolist()) == REORDERED


def test_reorder_refuses_pages_without_tokens():
    with pytest.raises(ValueError, match="at least one token"):
        eb.beam_reorder(*reorder_inputs((2, 12, 2, 0, 8), "cuda"))


def test_gradients_and_tangents_are_refused():
    check_gradients_are_refused("cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,new,dim", [(1030, 20, 64), (530, 300, 64), (1030, 20, 128)])
def test_attention_chunks_of_many_sequences(batch, new, dim, dtype):
    """More row tiles than the split's table holds: one item a CTA in the chunk kernel and the fp32 tiles."""
    lengths = [1 + (i * 53) % 450 for i in range(batch)]
    k, v, tables = make_cache(lengths, 1, dim, 32, dtype)
    positions = tail_positions(lengths, [min(n, new) for n in lengths], new)
    positions[11] = -1
    out = check_attention(queries(batch, new, 2, dim, dtype), k, v, tables, positions)
    assert not out[11].any()


def test_attention_record_names_the_kernel_that_ran():
    """Queries that are copied before the call are aligned, wherever the view began."""
    from exploration_b200.ops import launch
    k, v, tables = make_cache([90], 2, 64, 16, torch.bfloat16)
    base = torch.randn(2 * (1 * 40 * 8 * 64) + 1, device="cuda").to(torch.bfloat16)
    wide = base[1:].view(1, 40, 8, 128)[..., :64]
    assert wide.data_ptr() % 16 and not wide.is_contiguous()
    launch.reset()
    positions = tail_positions([90], [40], 40)
    out = eb.paged_attention(wide, k, v, tables, positions)
    assert torch.equal(out, eb.paged_attention(wide.contiguous(), k, v, tables, positions))
    [entry] = [e for e in launch.launch_report() if e["kernel"] == "paged_attention"]
    assert entry["calls"] == 2 and entry["path"] == "tcgen05"


@pytest.mark.parametrize("vocab", [50, 9000])
@pytest.mark.parametrize("new", [1, 40])
def test_a_whole_step_can_be_captured(new, vocab):
    """Append, attention, selection and reordering in one graph, replayed at other lengths."""
    torch.manual_seed(0)
    layers, groups, beams, heads, dim, page, width = 2, 2, 3, 4, 64, 16, 100
    pages = groups * beams * (width + 1)
    k, v = (torch.randn(layers, pages, heads, page, dim, device="cuda").to(torch.bfloat16) for _ in range(2))
    order = torch.randperm(pages, device="cuda").to(torch.int32).view(groups, beams, width + 1)
    tables, spare = order[..., :width].contiguous(), order[..., width].contiguous()
    qkv = torch.randn(layers, groups * beams, new, 3, heads, dim, device="cuda").to(torch.bfloat16)
    cos, sin = torch.rand(width * page, dim // 2, device="cuda"), torch.rand(width * page, dim // 2, device="cuda")
    logits, scores = torch.randn(groups, beams, vocab, device="cuda"), -torch.rand(groups, beams, device="cuda")
    ended = torch.zeros(groups, beams, dtype=torch.bool, device="cuda")
    lengths = torch.tensor([1200, 700], dtype=torch.int32, device="cuda")

    def step():
        last = lengths[:, None].expand(groups, beams).reshape(-1, 1)
        positions = last + torch.arange(new, device="cuda", dtype=torch.int32)
        outs = []
        for i in range(layers):
            q = eb.paged_append(*qkv[i].unbind(2), cos, sin, k[i], v[i], tables.flatten(0, 1), positions)
            outs.append(eb.paged_attention(q, k[i], v[i], tables.flatten(0, 1), positions))
        picked = eb.beam_select(logits, scores, ended, 3)
        moved = eb.beam_reorder(k, v, tables, spare, picked[1], lengths + new)
        return [*outs, *picked, *moved]

    start = k.clone(), v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for n in ([1200, 700], [16, 1], [1500, 1499]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        logits.normal_()
        results = []
        for run in (graph.replay, step):
            k.copy_(start[0])
            v.copy_(start[1])
            got = run()
            results.append([x.clone() for x in (got or captured)] + [k.clone(), v.clone()])
        assert all(torch.equal(a, b) for a, b in zip(*results))
