"""Decoding kernels at their edges, against their definitions in 64 bits (B200 only)."""
import pytest
import torch

import exploration_b200 as eb
from tests.test_paged_gpu import check_attention, make_cache, queries, tail_positions

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
