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
