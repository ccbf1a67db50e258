"""The ends of what the packed operators take: sizes of nothing, and outputs that must not be laid over other memory."""
import pytest
import torch

from conftest import announce
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("W", [1, 4])
def test_conv_without_channels(cuda, W):
    """There is nothing to compute, but the requests' status is told as ever."""
    from dforktree_amd import ops
    announce(f"prompt_conv without channels W={W}")
    x = torch.zeros(6, 0, dtype=BF16, device=cuda)
    state, weight = torch.zeros(2, 0, W - 1, dtype=BF16, device=cuda), torch.zeros(0, W, dtype=BF16, device=cuda)
    cu = torch.tensor([0, 3, 3, 6], dtype=torch.int32, device=cuda)
    status = torch.full((3,), -1, dtype=torch.int32, device=cuda)
    at = torch.tensor([1, -1, 2], device=cuda)
    y = ops.prompt_conv(x, state, weight, None, cu, max_len=2, cs_indices=at, status=status)
    assert y.shape == (6, 0) and status.tolist() == [P.STATUS_SPAN, 0, P.STATUS_SPAN | P.STATUS_SLOT]
    assert ops.prompt_conv(x, state, weight, batch=2).shape == (6, 0)
