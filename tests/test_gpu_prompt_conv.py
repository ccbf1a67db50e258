"""ops.prompt_conv against the 64-bit oracle.

Tolerance of an output: the sum of W products and the bias in 32 bits, (W + 1) 2^-24 of the sum of the terms' sizes; the
SiLU's slope is at most 1.1, its exp, sum and quotient 4 steps of 2^-24 of the value; then half a step of the output's
type.  Where all of x, weights and y are bf16 the exponential's argument z log2(e) is rounded to 2^-24 of itself: |z| 2^-24
of the value (at |z| = 88, past which fp32's exponential ends, 5 10^-6, beside bf16's half step of 4 10^-3).  A window is a copy: exact, or half a step of its type."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


def check(x, state, w, bias, cu, *, batch, limit, silu=True, indices=None, initial=None, y=None, cu_host=None, label=""):
    from dforktree_amd import ops
    announce(f"prompt_conv {label} x={tuple(x.shape)} {x.dtype} state={tuple(state.shape)} {state.dtype}")
    dev = x.device
    host = [t if t is None else t.double().cpu().numpy() for t in (x, state, w, bias)]
    want, want_state, want_status, size = P.prompt_conv(
        *host, cu_host, batch=batch, limit=limit, silu=silu, indices=None if indices is None else indices.tolist(),
        initial=None if initial is None else initial.tolist())
    status = torch.full((batch,), -1, dtype=torch.int32, device=dev)
    before = None if y is None else y.clone()
    y = ops.prompt_conv(x, state, w, bias, cu, max_len=limit, batch=None if cu is not None else batch, silu=silu,
                        cs_indices=indices, initial=initial, y=y, status=status)
    got = y.double().cpu().numpy()
    W = w.shape[1]
    tol = half_step(y.dtype) * np.abs(want) + 1.1 * (W + 1) * 2.0 ** -24 * size + 4 * 2.0 ** -24 * np.abs(want) + (
        2.0 ** -25 if y.dtype == F16 else 0)  # half of fp16's smallest step
    if x.dtype == w.dtype == y.dtype == BF16:
        tol += np.minimum(1.1 * size, 88) * 2.0 ** -24 * np.abs(want)  # |z| is at most the sum of the terms' sizes
    rows = ~np.isnan(want).any(1)
    bad = np.abs(got - want)[rows] > tol[rows]
    assert not bad.any(), (label, float(np.abs(got - want)[rows].max()))
    if before is not None:
        assert torch.equal(y[torch.tensor(~rows)], before[torch.tensor(~rows)])
    gs = state.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        near = np.abs(gs - want_state) <= half_step(state.dtype) * np.abs(want_state)
    same = (gs == want_state) | (np.isnan(gs) & np.isnan(want_state))
    assert same.all() if x.dtype == state.dtype else (near | same).all()
    assert status.tolist() == want_status.tolist()


def make(rows, C, W, slots, cuda, *, x=BF16, state=BF16, w=BF16, bias=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return (r(rows, C).to(x).to(cuda), r(slots, C, W - 1).to(state).to(cuda), (0.5 * r(C, W)).to(w).to(cuda),
            None if bias is None else r(C).to(bias).to(cuda))


def cu_of(sizes, cuda):
    host = [0, *np.cumsum(sizes).tolist()]
    return host, torch.tensor(host, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("sizes", [[1], [2], [3], [0, 1, 0, 4, 17], [15, 16, 17, 33], [100, 1, 64, 31, 32], [1] * 70])
@pytest.mark.parametrize("C", [8, 136, 2056])
def test_packed(cuda, sizes, C):
    host, cu = cu_of(sizes, cuda)
    B = len(sizes)
    x, s, w, b = make(sum(sizes), C, 4, B + 2, cuda, seed=C)
    at = torch.randperm(B + 2, generator=torch.Generator().manual_seed(B))[:B].to(cuda)
    init = torch.tensor([i % 3 != 1 for i in range(B)], device=cuda)
    check(x, s, w, b, cu, batch=B, limit=max(sizes), indices=at, initial=init, cu_host=host, label=str(sizes))


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("C", [1, 7, 264])
def test_widths(cuda, W, C):
    sizes = [5, 0, 1, W, 40]
    host, cu = cu_of(sizes, cuda)
    x, s, w, b = make(sum(sizes), C, W, 5, cuda, seed=W, bias=None)
    check(x, s, w, b, cu, batch=5, limit=40, silu=W % 2 == 0, cu_host=host, label=f"W={W}")


@pytest.mark.parametrize("x,state,w,y", [(BF16, F32, F32, F32), (F16, F16, F16, F16), (F32, BF16, F32, BF16),
                                         (BF16, BF16, F32, BF16), (F32, F32, F32, F32), (BF16, F16, BF16, F16)])
def test_types(cuda, x, state, w, y):
    sizes = [33, 1, 2, 18]
    host, cu = cu_of(sizes, cuda)
    t = make(sum(sizes), 72, 4, 4, cuda, x=x, state=state, w=w, bias=w, seed=3)
    out = torch.full((sum(sizes), 72), 7, dtype=y, device=cuda)
    check(*t, cu, batch=4, limit=33, y=out, cu_host=host, label=f"{x} {state} {w} {y}")


def test_strides(cuda):
    """Rows of a wider projection, windows kept channel last and with more columns, a transposed weight."""
    sizes = [20, 1, 3]
    host, cu = cu_of(sizes, cuda)
    x, s, w, b = make(24, 64, 4, 3, cuda, seed=5)
    wide = torch.randn(24, 200, device=cuda).bfloat16()
    wide[:, 33:97] = x
    last = torch.full((3, 5, 64), 9.0, device=cuda).bfloat16()
    last[:, :3] = s.transpose(1, 2)
    out = torch.zeros(24, 129, device=cuda).bfloat16()
    check(wide[:, 33:97], last.transpose(1, 2)[:, :, :3], w.t().contiguous().t(), b, cu, batch=3, limit=20,
          y=out[:, 1:65], cu_host=host, label="strides")
    assert (last[:, 3:] == 9).all() and not out[:, 0].any() and not out[:, 65:].any()


def test_wider_windows_keep_their_other_columns(cuda):
    x, s, w, b = make(10, 16, 4, 1, cuda, seed=6)
    wide = torch.full((1, 16, 6), 5.0, device=cuda).bfloat16()
    wide[:, :, :3] = s
    from dforktree_amd import ops
    ops.prompt_conv(x, wide, w, b)
    assert torch.equal(wide[0, :, :3], x[-3:].t()) and (wide[:, :, 3:] == 5).all()


@pytest.mark.parametrize("n", [1, 2, 37])
def test_uniform(cuda, n):
    x, s, w, b = make(6 * n + 2, 72, 4, 8, cuda, seed=n)
    out = torch.full(x.shape, 3.0, dtype=BF16, device=cuda)
    at = torch.tensor([3, -1, 0, 9, 7, 1], device=cuda)  # a padded request, one past the pool
    check(x, s, w, b, None, batch=6, limit=n, indices=at, y=out, label="uniform")


def test_cut_requests(cuda):
    """Longer than max_len, past the rows there are, and a first row that is not 0: the others keep their own."""
    x, s, w, b = make(50, 72, 4, 4, cuda, seed=8)
    for host in ([2, 12, 40, 41, 60], [0, 50, 50, 45, 50]):
        out = torch.full(x.shape, 3.0, dtype=BF16, device=cuda)
        cu = torch.tensor(host, dtype=torch.int32, device=cuda)
        check(x, s.clone(), w, b, cu, batch=4, limit=11, y=out, cu_host=host, label=str(host))


def test_not_finite_elsewhere(cuda):
    """Rows of no request and other requests' windows are never read."""
    x, s, w, b = make(30, 72, 4, 3, cuda, seed=9)
    x[20:] = float("nan")
    s[1] = float("inf")
    s[2] = float("nan")
    host, cu = [0, 10, 20], torch.tensor([0, 10, 20], dtype=torch.int32, device=cuda)
    check(x, s, w, b, cu, batch=2, limit=10, indices=torch.tensor([0, 2], device=cuda),
          initial=torch.tensor([True, False], device=cuda), y=torch.zeros(30, 72, device=cuda).bfloat16(), cu_host=host,
          label="not finite")


def test_offsets_past_32_bits(cuda):
    """Rows 2^24 elements apart and a window past 2^31 elements of the pool."""
    from dforktree_amd import ops
    announce("prompt_conv offsets past 32 bits")
    T, C = 140, 16
    x, s, w, b = make(T, C, 4, 1, cuda, seed=10)
    far = torch.empty(T << 24, dtype=BF16, device=cuda).as_strided((T, C), (1 << 24, 1)).copy_(x)
    pool = torch.empty((1 << 31) + 64, dtype=BF16, device=cuda).as_strided((2, C, 3), (1 << 31, 3, 1))
    pool.copy_(s.expand(2, C, 3))
    y = ops.prompt_conv(far, pool, w, b, cs_indices=torch.tensor([1], device=cuda))
    near = s.clone()
    assert torch.equal(y, ops.prompt_conv(x, near, w, b))
    assert torch.equal(pool[1], near[0]) and torch.equal(pool[0], s[0])


def test_captured_and_on_another_stream(cuda):
    """A captured decode step goes on from where the last replay ended; the launch is on the current stream."""
    from dforktree_amd import ops
    announce("prompt_conv in a graph")
    x, s, w, b = make(6, 72, 4, 6, cuda, seed=11)
    eager, y = s.clone(), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_conv(x, s.clone(), w, b, max_len=1, batch=6, y=y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_conv(x, s, w, b, max_len=1, batch=6, y=y)
    for step in range(4):
        x.copy_(torch.randn(6, 72, generator=torch.Generator().manual_seed(step)))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.prompt_conv(x, eager, w, b, max_len=1, batch=6)
        assert torch.equal(y, want) and torch.equal(s, eager)


def test_refused(cuda):
    from dforktree_amd import ops
    x, s, w, b = make(6, 16, 4, 2, cuda)
    for kw, err in ((dict(x=x.t()), ValueError), (dict(weight=w[:8]), ValueError), (dict(bias=b[:8]), ValueError),
                    (dict(conv_state=s[:, :, :2]), ValueError), (dict(conv_state=s[0]), ValueError),
                    (dict(y=x), ValueError), (dict(y=x[:3]), ValueError), (dict(x=x.int()), TypeError),
                    (dict(cs_indices=torch.zeros(3, dtype=torch.int32, device=cuda)), ValueError),
                    (dict(cs_indices=torch.zeros(1, device=cuda)), TypeError),
                    (dict(initial=torch.zeros(1, device=cuda)), TypeError),
                    (dict(initial=torch.zeros(2, dtype=torch.bool, device=cuda)), ValueError),
                    (dict(conv_state=s[:1].expand(2, -1, -1)), ValueError), (dict(max_len=2, batch=4), ValueError),
                    (dict(conv_state=s, max_len=2, batch=3), ValueError), (dict(conv_state=s.cpu()), ValueError),
                    (dict(cu_seqlens=torch.tensor([0, 6], device=cuda)), TypeError),
                    (dict(cu_seqlens=torch.tensor([0, 6], dtype=torch.int32, device=cuda)), ValueError)):
        with pytest.raises(err):
            ops.prompt_conv(**(dict(x=x, conv_state=s, weight=w, bias=b) | kw))
    # nothing to do
    assert ops.prompt_conv(x[:0], s, w, b, max_len=0, batch=2).shape == (0, 16)
