"""ops.tree_accept where the running sum meets its target at the border of parts without any weight, as rows have them
that were cut to their likeliest tokens."""
import numpy as np
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,at,rows,calls", [
    (8, [0, 1, 2, 4, 5, 6], 40000, 1),                                   # a part of one token each, by one workgroup
    (4000, [100, 700, 1200, 2100, 2600, 3100], 2000, 15),                # parts of 500
    (20480, [100, 1124, 2148, 10245, 11269, 12293], 100, 300),           # slices of 1024
    (100003, [5, 2100, 4200, 50005, 52100, 54200], 30, 500)])            # slices of 2048
def test_half_of_a_row_of_two_like_halves(cuda, V, at, rows, calls):
    """Half of the sum is the border behind the third of six weights: the token is the third or the fourth of them, by the
    roundings of 64-bit sums, and never one of the parts between them, which have none."""
    from dforktree_amd import ops
    announce(f"tree_accept at a border V={V}")
    rng = np.random.default_rng(V)
    zero = torch.zeros(rows, dtype=torch.int32, device=cuda)
    u, half = torch.zeros(rows, device=cuda), torch.full((rows,), 0.5, device=cuda)
    p = torch.zeros(rows, V, device=cuda)
    for _ in range(calls):
        w = np.exp(rng.normal(0, 8, (rows, 3))).astype(np.float32)
        p[:, at] = torch.from_numpy(np.concatenate([w, w], 1)).to(cuda)
        status = torch.full((rows,), -1, dtype=torch.int32, device=cuda)
        token = ops.tree_accept(zero, zero, p, u, half, n_nodes=1, batch=rows, status=status)["token"]
        assert not status.any() and (token >= 0).all()
        place = np.searchsorted(at, token.cpu().numpy())
        assert np.array_equal(np.array(at)[place], token.cpu().numpy())
        # the sum up to the token, and in front of it, beside half of the whole
        run, want = np.cumsum(np.concatenate([w, w], 1).astype(np.float64), 1), w.astype(np.float64).sum(1)
        upto = np.take_along_axis(run, place[:, None], 1)[:, 0]
        before = np.where(place, np.take_along_axis(run, np.maximum(place - 1, 0)[:, None], 1)[:, 0], 0)
        assert (before <= want * (1 + 2.0 ** -48)).all() and (upto >= want * (1 - 2.0 ** -48)).all()
