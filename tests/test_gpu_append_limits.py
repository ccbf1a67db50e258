"""kv_append at the ends of its ranges."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 64), (1, 5)])
def test_no_source_rows(cuda, shape):
    """An entry that names a row of none is one past the rows: skipped and marked."""
    from dforktree_amd import ops
    announce(f"append without rows {shape}")
    k = torch.empty(0, *shape, device=cuda)
    cache = torch.full((3, 4, *shape), 5.0, device=cuda)
    for slots, rows, word in (([3, 4], [0, -1], 1), ([-1, 4], [0, -1], 0)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        ops.kv_append(k, k, cache, cache.clone(), torch.tensor(slots, device=cuda), rows=torch.tensor(rows, device=cuda), status=status)
        torch.cuda.synchronize()
        assert status.item() == word and (cache == 5).all()


@pytest.mark.parametrize("src", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dst", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("heads,d", [(4, 64), (3, 7)])
def test_every_cast(cuda, src, dst, heads, d):
    """Rounded once, to the nearest and ties to even; past fp16's range infinity; NaN stays NaN."""
    from dforktree_amd import ops
    announce(f"append cast {src}->{dst} {heads}x{d}")
    src, dst = getattr(torch, src), getattr(torch, dst)
    g = torch.Generator().manual_seed(d)
    bits = torch.randint(-2 ** 31, 2 ** 31, (70, 2, heads, d), generator=g).to(torch.int32)
    x = bits.view(torch.float32) if src == torch.float32 else (bits >> 16).to(torch.int16).view(src)
    x[:20] = torch.randn(20, 2, heads, d, generator=g).to(src)
    x[0, :, 0, :4] = torch.tensor([0.0, -0.0, float("inf"), -float("inf")]).to(src)
    slots = torch.randperm(80, generator=g)[:70]
    caches = [torch.zeros(5, 16, heads, d, dtype=dst, device=cuda) for _ in range(2)]
    y = x.to(cuda)
    ops.kv_append(y[:, 0], y[:, 1], *caches, slots.to(cuda))
    torch.cuda.synchronize()
    for cache, new in zip(caches, (x[:, 0], x[:, 1])):
        got, want = cache.cpu().view(80, heads, d)[slots], new.to(dst)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(torch.signbit(got) | nan, torch.signbit(want) | nan)
        assert torch.equal(got[~nan], want[~nan])


def test_moves_within_a_cache(cuda):
    """Rows may be the cache's own slots where none that is read is written, or only by itself."""
    from dforktree_amd import ops
    announce("append within a cache")
    g = torch.Generator().manual_seed(2)
    caches = [torch.randn(6, 16, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2)]
    order = torch.randperm(96, generator=g)
    rows, slots = order[:40].clone(), order[40:80].clone()
    rows[:5] = slots[:5]
    want = [c.clone().view(96, 2, 64) for c in caches]
    for w in want:
        w[slots] = w[rows]
    x = [c.to(cuda) for c in caches]
    ops.kv_append(x[0].view(96, 2, 64), x[1].view(96, 2, 64), *x, slots.to(cuda), rows=rows.to(cuda))
    torch.cuda.synchronize()
    for c, w in zip(x, want):
        assert torch.equal(c.cpu().view(96, 2, 64), w)
