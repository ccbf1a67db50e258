"""Paged attention where items are cut and shares hold many, and caches without pages; prompts in large batches."""
import numpy as np
import pytest
import torch

from conftest import announce
from test_gpu_attention import BF16, F16, Paged, ancestry, check_prompt, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [257, 700])
def test_more_requests_than_threads(cuda, batch):
    """Several requests a thread in the scan of the shares, empty ones among them."""
    announce(f"{batch} requests")
    rng = np.random.default_rng(batch)
    prefix = rng.integers(0, 90, batch).tolist()
    new = [int(x) for x in rng.integers(0, 3, batch)]
    prefix[batch // 2] = 700  # a table past what is never cut
    t = Paged(cuda, 1, prefix, new, hq=4, hkv=2, d=64, ps=8)
    t.check(*t.run(), what=f"{batch} requests")


@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, F16), (256, BF16)])
@pytest.mark.parametrize("causal", [True, False])
def test_many_row_tiles(cuda, d, dtype, causal):
    """Items of one request side by side on a line, more parts than waves of the join."""
    announce(f"row tiles d={d} {dtype} causal={causal}")
    t = Paged(cuda, d, [900, 0, 3000, 40], [333, 70, 40, 1], hq=8, hkv=1, d=d, ps=24, dtype=dtype)
    t.check(*t.run(causal=causal), causal=causal, what=f"row tiles d={d}")


def test_long_trees(cuda):
    """A tree's item in more than eight parts."""
    announce("long trees")
    bits = ancestry([64, 20], 1)
    t = Paged(cuda, 3, [6000, 900], [64, 20], hq=8, hkv=2, d=128, ps=16)
    t.check(*t.run(bits=bits), bits=bits, what="long trees")


@pytest.mark.parametrize("pages,columns", [(0, 0), (0, 5), (3, 0), (0, 700)])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_nothing_to_read(cuda, pages, columns, rows):
    """No pages, or a table without columns: no keys, whatever the lengths say."""
    from dforktree_amd import ops
    announce(f"pages={pages} columns={columns} rows={rows}")
    cache = torch.full((pages, 16, 2, 128), float("nan"), dtype=BF16, device=cuda)
    q = torch.randn(2 * rows, 8, 128, device=cuda).to(BF16)
    lse = torch.zeros(2 * rows, 8, device=cuda)
    o = ops.paged_attention(q, cache, cache, torch.zeros(2, columns, dtype=torch.int32, device=cuda),
                            torch.tensor([9, 4000], device=cuda), n_new=rows, lse=lse)
    torch.cuda.synchronize()
    assert (o == 0).all() and (lse == -np.inf).all()


@pytest.mark.parametrize("batch", [2, 63, 64, 65, 90])
def test_batches_of_prompts(cuda, batch):
    """Both orders of the items; lengths that repeat, and none."""
    announce(f"{batch} prompts")
    rng = np.random.default_rng(batch)
    sizes = [int(x) for x in rng.integers(0, 150, batch)]
    sizes[0], sizes[-1] = 260, 0
    r = prompt(cuda, sizes, 4, 2, 64, BF16, seed=batch)
    check_prompt(*r, sizes, 4, 2, 64, BF16, what=f"{batch} prompts")
    r = prompt(cuda, [97] * batch, 4, 2, 64, BF16, seed=batch)
    check_prompt(*r, [97] * batch, 4, 2, 64, BF16, what=f"{batch} equal prompts")


def test_prompts_with_nothing(cuda):
    """A packed batch of empty prompts writes its status words and nothing else."""
    from dforktree_amd import ops
    announce("empty prompts")
    x = torch.randn(7, 8, 64, device=cuda).to(BF16)
    o, status = torch.full((7, 4, 64), 3.0, dtype=BF16, device=cuda), torch.full((3,), 9, dtype=torch.int32, device=cuda)
    ops.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], torch.tensor([0, 0, 0, 0], dtype=torch.int32, device=cuda), max_len=7,
                         o=o, status=status)
    torch.cuda.synchronize()
    assert (o == 3).all() and status.tolist() == [0, 0, 0]
