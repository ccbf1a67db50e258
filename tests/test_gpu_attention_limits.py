"""Paged and prompt attention where a request is cut, no row is left, rows belong to nobody, or the launch's bounds are far
above the work."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P
from test_gpu_attention import BF16, Paged, ancestry, check, check_prompt, dense, prompt

pytestmark = pytest.mark.gpu


def ints(cuda, x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kept", [2, 9])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("far", [90, 900])
def test_a_cut_request_keeps_its_first_rows(cuda, d, kept, tree, far):
    """They see what they see in the whole request: the rows that are left out still stand behind them."""
    from dforktree_amd import _lib, ops
    announce(f"cut to {kept} rows d={d} tree={tree} prefix={far}")
    sizes = [2, 40, 1]
    t = Paged(cuda, d, [30, far, 70], sizes, hq=8, hkv=2, d=d, ps=16)
    bits = ancestry(sizes, 4) if tree else None
    k, v = t.caches()
    o = torch.full(t.q.shape, 7.0, dtype=BF16, device=cuda)
    lse, status = torch.full(t.q.shape[:2], 7.0, device=cuda), ints(cuda, [9] * 3)
    ops.paged_attention(t.gpu(t.q), k, v, t.gpu(t.table), ints(cuda, t.total), cu_seqlens=t.gpu(t.cu), n_new=kept, o=o, lse=lse,
                        anc_bits=None if bits is None else t.gpu(bits), status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, _lib.DFT_STATUS_SPAN, 0]
    assert (o[2 + kept:42] == 7).all() and (lse[2 + kept:42] == 7).all()
    for b, n in enumerate(sizes):
        r0, L, m = int(t.cu[b]), t.total[b], min(n, kept)
        sees = (P.sees_tree(bits[r0:r0 + n].numpy(), L) if tree else P.sees_causal(n, L))[:m]
        keys, values = (torch.as_tensor(P.paged_keys(c.float().numpy(), t.table[b].numpy(), L)[0]).double() for c in (t.k, t.v))
        r = slice(r0, r0 + m)
        check(o[r], lse[r], dense(t.q[r].double(), keys, values, sees, d ** -0.5), L, BF16, 10.0, f"request {b}")


def test_status_without_rows(cuda):
    """The status words are written also where there is no row to write."""
    from dforktree_amd import _lib, ops
    announce("status without rows")
    SPAN, TABLE = _lib.DFT_STATUS_SPAN, _lib.DFT_STATUS_TABLE
    x = torch.zeros(4, 4, 64, dtype=BF16, device=cuda)
    cache = torch.zeros(3, 16, 2, 64, dtype=BF16, device=cuda)
    for rows, limit, cu, want in ((4, 0, [0, 0, 3], [0, SPAN]), (0, 3, [0, 0, 3], [0, SPAN]), (0, 0, [0, 0, 0], [0, 0]),
                                  (4, 0, [2, 1, 1], [SPAN, 0])):
        for columns, extra in ((2, TABLE), (40, 0)):
            status = ints(cuda, [99, 99])
            ops.paged_attention(x[:rows], cache, cache, torch.zeros(2, columns, dtype=torch.int32, device=cuda),
                                ints(cuda, [5, 100]), cu_seqlens=ints(cuda, cu), n_new=limit, status=status)
            torch.cuda.synchronize()
            assert status.tolist() == [want[0], want[1] | extra], (rows, limit, cu, columns)
        status = ints(cuda, [99, 99])
        ops.prompt_attention(x[:rows], x[:rows, :2], x[:rows, :2], ints(cuda, cu), max_len=limit, status=status)
        torch.cuda.synchronize()
        assert status.tolist() == want, (rows, limit, cu)
    status = ints(cuda, [99, 99])
    ops.paged_attention(x[:0], cache, cache, torch.zeros(2, 2, dtype=torch.int32, device=cuda), ints(cuda, [5, 100]),
                        status=status)  # without cu_seqlens
    torch.cuda.synchronize()
    assert status.tolist() == [0, TABLE]


def test_bounds_far_above_the_rows(cuda):
    """n_new is a bound: short rows under a long one are served."""
    from dforktree_amd import ops
    announce("far bounds")
    rng = np.random.default_rng(0)
    prefix, new = [int(x) for x in rng.integers(0, 60, 300)], [int(x) for x in rng.integers(0, 4, 300)]
    t = Paged(cuda, 0, prefix, new, hq=1, hkv=1, d=64, ps=16)
    k, v = t.caches()
    lse = torch.empty(t.rows, 1, device=cuda)
    o = ops.paged_attention(t.gpu(t.q), k, v, t.gpu(t.table), ints(cuda, t.total), cu_seqlens=t.gpu(t.cu), n_new=1 << 23, lse=lse)
    torch.cuda.synchronize()
    t.check(o, lse, what="paged")


def test_prompt_bounds_far_above_the_rows(cuda):
    """max_len is a bound: short prompts under a long one are served."""
    from dforktree_amd import ops
    announce("far bounds of prompts")
    rng = np.random.default_rng(0)
    sizes = [int(x) for x in rng.integers(0, 60, 100)]
    qkv, want, lse = prompt(cuda, sizes, 4, 4, 64, BF16)
    check_prompt(qkv, want, lse, sizes, 4, 4, 64, BF16, what="prompts")
    x = qkv.to(cuda)
    o = ops.prompt_attention(x[:, :4], x[:, 4:8], x[:, 8:], ints(cuda, [0, *np.cumsum(sizes)]), max_len=1 << 24)
    torch.cuda.synchronize()
    assert torch.equal(o, want)


def test_one_long_prompt_among_very_many(cuda):
    """More row tiles (of the longest, for every prompt) than one launch can count."""
    from dforktree_amd import ops
    announce("one long prompt among 65535")
    B, n, hq, hkv, d = 65535, 1100, 32, 8, 64
    sizes = np.ones(B, int)
    sizes[B - 3] = n
    cu = ints(cuda, [0, *np.cumsum(sizes)])
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn(int(sizes.sum()), h, d, generator=g, device=cuda).to(BF16) for h in (hq, hkv, hkv))
    status = torch.full((B,), 9, dtype=torch.int32, device=cuda)
    o = ops.prompt_attention(q, k, v, cu, max_len=n, status=status)
    torch.cuda.synchronize()
    assert not status.any()
    r = slice(B - 3, B - 3 + n)
    assert torch.equal(o[r], ops.prompt_attention(q[r], k[r], v[r]))
    alone = torch.ones(q.shape[0], dtype=torch.bool, device=cuda)
    alone[r] = False
    assert torch.equal(o[alone], v[alone].repeat_interleave(hq // hkv, 1))  # one token sees itself


def test_rows_of_no_request_are_not_written(cuda):
    """Rows past the last request (a captured step's padding) keep what they hold."""
    from dforktree_amd import ops
    announce("padding rows")
    t = Paged(cuda, 1, [20, 700], [3, 4], hq=8, hkv=2, d=64, ps=16)
    q = torch.cat([t.q, torch.full((5, 8, 64), float("nan"), dtype=BF16)]).to(cuda)
    k, v = t.caches()
    for n_new, width in ((4, None), (40, None), (4, 32)):
        o, lse = torch.full(q.shape, 7.0, dtype=BF16, device=cuda), torch.full(q.shape[:2], 7.0, device=cuda)
        ops.paged_attention(q, k, v, t.gpu(t.table)[:, :width], ints(cuda, t.total), cu_seqlens=t.gpu(t.cu), n_new=n_new, o=o,
                            lse=lse)
        torch.cuda.synchronize()
        assert (o[7:] == 7).all() and (lse[7:] == 7).all() and torch.isfinite(o).all()
        if width is None:
            t.check(o, lse, what=f"n_new={n_new}")
    x = torch.randn(12, 8, 64, device=cuda).to(BF16)
    o = torch.full((12, 4, 64), 7.0, dtype=BF16, device=cuda)
    ops.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], ints(cuda, [0, 3, 7]), max_len=6, o=o)
    torch.cuda.synchronize()
    assert (o[7:] == 7).all() and not (o[:7] == 7).all(-1).any()


@pytest.mark.parametrize("new", [[1, 20], [1, 3]])
def test_far_interleaved_caches(cuda, new):
    """Keys and values as every other page of one buffer, with a page stride past 2^31 elements."""
    from dforktree_amd import ops
    announce(f"far interleaved caches {new}")
    t = Paged(cuda, 14, [10, 15], new, hq=8, hkv=2, d=128, ps=16, poison=False)
    pages, page = t.k.shape[0], 16 * 2 * 128
    step = (1 << 31) + 4 * page
    buffer = torch.empty((pages - 1) * step + 2 * page, dtype=BF16, device=cuda)
    k, v = (torch.as_strided(buffer, (pages, 16, 2, 128), (step, 256, 128, 1), at) for at in (0, page))
    k.copy_(t.gpu(t.k))
    v.copy_(t.gpu(t.v))
    lse = torch.empty(t.q.shape[:2], device=cuda)
    o = ops.paged_attention(t.gpu(t.q), k, v, t.gpu(t.table), ints(cuda, t.total), cu_seqlens=t.gpu(t.cu), n_new=max(new), lse=lse)
    t.check(o, lse, what="interleaved")
    del buffer, k, v
    torch.cuda.empty_cache()
