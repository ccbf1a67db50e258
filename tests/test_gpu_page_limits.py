"""Page plans at the ends of their ranges."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P
from test_gpu_pages import compare, tables

pytestmark = pytest.mark.gpu

TOP = 2 ** 63 - 1


@pytest.mark.parametrize("ps", [1, 16, 2 ** 31 - 1])
@pytest.mark.parametrize("batch", [5, 300])
def test_lengths_of_any_size(cuda, ps, batch):
    """64-bit lengths whose sums would leave 64 bits: too many tokens for the table or the rows, and nothing else."""
    announce(f"lengths of any size page={ps} batch={batch}")
    prefix, new = [3, 2 ** 62, TOP, -TOP - 1, 7], [2, 1, 0, 3, 0]
    want = [0, P.STATUS_TABLE, P.STATUS_TABLE, P.STATUS_SPAN, 0]
    if batch == 300:
        prefix, new = prefix * 60, new * 60
        want = want * 60
    B = len(prefix)
    free = np.arange(40 * B, dtype=np.int32)
    table = np.full((B, 30), -1, np.int32)
    r = compare(cuda, prefix, new, table, [0] * B, free, [9, 9 + len(free)], ps=ps, rows=sum(new), index=torch.int64, trim=True)
    assert r["status"].tolist() == want
    new = [2, TOP, TOP, -TOP - 1, TOP]
    r = compare(cuda, [0, 1, 5, 2, 3], new, table[:5], [0] * 5, free, [9, 9 + len(free)], ps=max(ps, 16), rows=12, index=torch.int64)
    assert r["cu_seqlens"].tolist() == [0, 2, 12, 12, 12, 12] and r["status"].tolist() == [0, 1, 1, 1, 1]


@pytest.mark.parametrize("batch", [4097, 8192])
def test_largest_batches(cuda, batch):
    """Running sums in more LDS than a launch has without asking, up to the limit."""
    announce(f"plan of {batch} requests")
    rng = np.random.default_rng(batch)
    prefix, new = rng.integers(0, 60, batch), rng.integers(0, 9, batch)
    held = -(-prefix // 4) + rng.integers(0, 3, batch)
    table, free = tables(rng, held, 25, 2 * batch)
    head = 11
    ring = np.full(int(sum(held)) + len(free), -1, np.int32)
    ring[(head + np.arange(len(free))) % len(ring)] = free
    for trim in (False, True):
        compare(cuda, prefix, new, table, held, ring, [head, head + len(free)], ps=4, rows=int(new.sum()), trim=trim,
                depth=rng.integers(0, 9, int(new.sum())))
