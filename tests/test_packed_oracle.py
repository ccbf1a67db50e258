"""The 64-bit oracle of the operators around the tree step: against closed forms, and the accepted tokens' distribution
by enumeration of what the random numbers decide."""
import itertools

import numpy as np
import pytest

from oracle import gdn_tree as O
from oracle import packed as P


def test_conv_of_a_whole_prompt_is_numpy_convolution():
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((9, 3)), rng.standard_normal((3, 4))
    y, state, status, _ = P.prompt_conv(x, np.zeros((1, 3, 3)), w, None, None, batch=1, limit=9, silu=False)
    for c in range(3):
        assert np.allclose(y[:, c], np.convolve(x[:, c], w[c, ::-1])[:9])
    assert np.array_equal(state[0], x[-3:].T) and not status.any()


def test_conv_in_pieces_is_the_whole():
    rng = np.random.default_rng(1)
    x, w, s0 = rng.standard_normal((10, 2)), rng.standard_normal((2, 4)), rng.standard_normal((1, 2, 3))
    whole = P.prompt_conv(x, s0, w, None, None, batch=1, limit=10)
    state, parts = s0, []
    for i, j in ((0, 1), (1, 3), (3, 10)):
        y, state, _, _ = P.prompt_conv(x[i:j], state, w, None, None, batch=1, limit=j - i)
        parts.append(y)
    assert np.allclose(np.concatenate(parts), whole[0]) and np.allclose(state, whole[1])


def test_gdn_rows_are_a_chain_of_tree_nodes():
    """The tree oracle (pinned against the reference's formulas) over a chain gives the same rows."""
    rng = np.random.default_rng(2)
    N, hk, hv = 16, 1, 2
    y = O.bf16_round(rng.standard_normal((1, N, (2 * hk + hv) * 128)))
    a, b = rng.standard_normal((2, 1, N, hv)).astype(np.float32)
    A_log, dt = rng.standard_normal(hv).astype(np.float32), rng.standard_normal(hv).astype(np.float32)
    S0 = (0.05 * rng.standard_normal((1, hv, 128, 128))).astype(np.float32)
    anc = np.tril(np.ones((1, N, N), np.float32))
    ref = O.tree_gdn_split(y, a, b, A_log, dt, S0, anc, hk, hv, 128, 128)
    o, _, _ = P.prompt_gdn(y[0], a[0], b[0], -np.exp(A_log), dt, S0, None, hk=hk, hv=hv, batch=1, limit=N)
    assert np.linalg.norm(ref["o"][0] - o) / np.linalg.norm(o) < 1e-5


@pytest.mark.parametrize("drawn", [False, True])
def test_accepted_tokens_follow_the_target(drawn):
    """A root with two children, 4 tokens: the first token behind the root is distributed as the target's row, over a fine
    grid of all random numbers (and, where the drafter draws, over all ordered pairs of its children).

    A grid of m midpoints per number is off by at most one cell per border: 4 borders in the last number, one in each
    of the two tests, so 6 / m per token."""
    p = np.array([0.1, 0.2, 0.3, 0.4])
    q = np.array([0.4, 0.3, 0.2, 0.1])
    m = 24
    grid = (np.arange(m) + 0.5) / m
    pairs = list(itertools.permutations(range(4), 2)) if drawn else [(1, 0)]
    got = np.zeros(4)
    for i, j in pairs:
        share = q[i] * q[j] / (1 - q[i]) if drawn else 1.0
        for u1, u2, last in itertools.product(grid, grid, grid):
            probs = np.stack([p] * 3)
            path, token = P.accept([9, i, j], [-1, 0, 0], probs, [0, u1, u2], last, np.stack([q] * 3) if drawn else None)
            first = [9, i, j][path[1]] if len(path) > 1 else token
            got[first] += share / m ** 3
    assert abs(got.sum() - 1) < 1e-9 and np.abs(got - p).max() < 6 / m


def test_accept_walks_the_tree():
    V = 5
    probs = np.full((5, V), 0.2)
    # 0 -> 1 -> 3, 0 -> 2 -> 4; u = 0 always stands, u = 0.99 never
    parent, tokens = [-1, 0, 0, 1, 2], [0, 1, 2, 3, 4]
    assert P.accept(tokens, parent, probs, [0, 0, 0, 0, 0], 0.5)[0] == [0, 1, 3]
    assert P.accept(tokens, parent, probs, [0, .99, 0, 0, 0], 0.5)[0] == [0, 2, 4]
    assert P.accept(tokens, parent, probs, [0, .99, .99, 0, 0], 0.0) == ([0], 0)  # of 0, 3 and 4
    assert P.accept(tokens, parent, probs, [0, .99, .99, 0, 0], 0.4) == ([0], 3)
    assert P.accept(tokens, parent, probs, [0, 0, 0, 0, 0], 0.5, path_cols=2) == ([0, 1], 2)
    assert P.accept(tokens, parent, probs * 0, [0, 0, 0, 0, 0], 0.5) == ([0], -1)
