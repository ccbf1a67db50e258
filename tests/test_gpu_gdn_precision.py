"""ops.prompt_gdn in 32 bits: states and fp32 outputs as near to the 64-bit recurrence as 32 bits allow.

Tolerance.  Three bf16 parts hold a factor to 2^-24 of itself, as 32 bits do, and a product of two such factors leaves
out 2 * 2^-24.  Between a row's inputs and the state stand: k's norm (its sum, root and quotient: 3 roundings), the
decay (its exponent's product and sum, its exponential: 3), beta (2), S in parts, the sum over the keys and its decay
(3), v less that (1), W and X in parts with the product of the two (4), so 16 of 2^-24 in the 2-norm each; what a write
adds is rounded once more per chunk, where a row's write is a contraction (beta <= 1, |k| = 1) and passes an earlier
error on at most whole, as its share of the state.  Roundings of many elements do not point one way: their sum in the
2-norm is below the sum of their bounds, and those of later chunks stand beside it.  So the state is held to 16 * 2^-24.
An output has q's norm (3) and the sum of its two products (1) on top: 20 * 2^-24.  (A two-part factor anywhere is off
by 2^-16 at most and by 4 10^-6 or so in the 2-norm.)"""
import numpy as np
import pytest
import torch

from conftest import announce, rel_l2
from oracle import packed as P
from test_gpu_gdn import F32, Case, cu_of

pytestmark = pytest.mark.gpu

STATE, OUT = 16 * 2.0 ** -24, 20 * 2.0 ** -24


def check(c, sizes, cuda, *, label="", o_dtype=F32, state=None):
    """The outputs and states of c's packed requests, each from its slot."""
    from dforktree_amd import ops
    host, cu = cu_of(sizes, cuda)
    announce(f"prompt_gdn in 32 bits {label} {len(sizes)} requests, {host[-1]} rows, {c.hk} and {c.hv} heads")
    state = c.pool.transpose(-1, -2) if state is None else state
    h = lambda t: t.double().cpu().numpy()  # noqa: E731
    rate = -torch.exp(c.A_log.float())
    want, want_state, _ = P.prompt_gdn(h(c.y), h(c.a), h(c.b), h(rate), h(c.dt_bias), h(state), host, hk=c.hk, hv=c.hv,
                                       batch=len(sizes), limit=max(sizes))
    o = ops.prompt_gdn(c.y, c.a, c.b, None, c.dt_bias, state, cu, hk=c.hk, hv=c.hv, max_len=max(sizes),
                       neg_exp_A=rate.contiguous(), o_dtype=o_dtype)
    got, half = h(o), torch.finfo(o_dtype).eps / 2
    for b, (i, j) in enumerate(zip(host, host[1:])):
        if i == j:
            continue
        assert rel_l2(h(state[b]), want_state[b]) <= STATE, (label, b, rel_l2(h(state[b]), want_state[b]))
        if o_dtype == F32:
            assert rel_l2(got[i:j], want[i:j]) <= OUT, (label, b, rel_l2(got[i:j], want[i:j]))
        else:
            tol = half * np.abs(want[i:j]) + 2.0 ** -19 * np.abs(want[i:j]).max()
            assert (np.abs(got[i:j] - want[i:j]) <= tol).all(), (label, b)
    return o


@pytest.mark.parametrize("sizes", [[64], [130], [17, 65, 200], [1000], [100] * 40])
@pytest.mark.parametrize("hk,hv", [(1, 1), (2, 8)])
def test_weak_gates(cuda, sizes, hk, hv):
    """Chunks with 16 and with 32 value columns a workgroup."""
    c = Case(sum(sizes), hk, hv, len(sizes), cuda, seed=sum(sizes), gates=F32, decay=0.02)
    check(c, sizes, cuda, label="weak gates")


def strong(c, at, g):
    """Rows `at` with the log decay g among weak ones, through softplus's inverse."""
    gen = torch.Generator().manual_seed(len(at))
    weak = 1e-3 + 0.02 * torch.rand(c.a.shape, generator=gen, dtype=torch.float64)
    a = torch.log(torch.expm1(weak))
    a[at] = -g
    c.a = a.float().to(c.y.device)
    c.A_log, c.dt_bias = torch.zeros(c.hv, device=c.y.device), torch.zeros(c.hv, device=c.y.device)


@pytest.mark.parametrize("sizes", [[64], [200], [30, 100, 64]])
@pytest.mark.parametrize("g", [-30.0, -100.0, -300.0, -4000.0, float("-inf")])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.4, 0.75])
def test_resets_among_weak_gates(cuda, sizes, g, share):
    """Rows that leave nothing of the state, one of them or some of every chunk: what the weak gates behind them keep is as
    exact as without them."""
    n = sum(sizes)
    c = Case(n, 1, 2, len(sizes), cuda, seed=n, gates=F32)
    at = torch.randperm(n, generator=torch.Generator().manual_seed(n))[:max(1, int(share * n))]
    strong(c, at, g)
    check(c, sizes, cuda, label=f"{len(at)} rows of g={g}")


@pytest.mark.parametrize("sizes", [[64], [130], [20, 300, 65], [1000], [100] * 40])
@pytest.mark.parametrize("decay", [0.3, 1.0, 30.0, 1000.0])
def test_ordinary_and_strong_gates(cuda, sizes, decay):
    c = Case(sum(sizes), 2, 8, len(sizes), cuda, seed=sum(sizes) + 1, gates=F32, decay=decay)
    check(c, sizes, cuda, label=f"decay {decay}")
