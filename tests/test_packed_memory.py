"""Which outputs of the packed operators are refused for the memory that they lie over, against the sets of elements."""
import random

import torch


def test_outputs_over_their_own_or_the_inputs_rows():
    from dforktree_amd.ops import _own_memory
    rng, index = random.Random(0), torch.arange(400)
    seen = {}
    for _ in range(6000):
        pitch = rng.choice((8, 10, 13))
        x = index.as_strided((rng.randint(1, 5), rng.randint(1, 8)), (pitch, 1), rng.randint(0, 60))
        other = rng.choice((pitch, pitch, pitch, 11))
        if rng.random() < 0.5:
            out = index.as_strided((rng.randint(1, 5), rng.randint(1, 8)), (other, 1), rng.randint(0, 80))
        else:
            shape = rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 4)
            out = index.as_strided(shape, (other, rng.choice((4, 5, 40)), 1), rng.randint(0, 80))
        at = out.flatten().tolist()
        alone = len(set(at)) == len(at) and not set(at) & set(x.flatten().tolist())
        try:
            _own_memory(out, "out", x, "x")
            refused = False
        except ValueError as e:
            assert "must not lie over" in str(e)
            refused = True
        assert not (refused and alone), (x.shape, x.stride(), out.shape, out.stride())
        if out.dim() == 2 and other == pitch:  # rows of one pitch: every overlap is seen
            assert refused != alone, (x.shape, x.stride(), out.shape, out.stride())
        seen[refused] = seen.get(refused, 0) + 1
    assert min(seen.values()) > 500
