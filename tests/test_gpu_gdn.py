"""ops.prompt_gdn and ops.token_gdn against the 64-bit recurrence.

Tolerances.  A factor that is held as a bf16 pair is off by at most 2^-8 * 2^-8 = 2^-16 relative, a product of two such
pairs leaves out lo * lo, another 2^-16; sums, decays and gates are in 32 bits.  u goes through two such products (S^T k
and X w), the state through one more (k u^T), o through four.  The write is a contraction (beta <= 1, |k| <= 1), so what a
row gets wrong does not grow from row to row; errors of rows add up at most as the rows' shares of the state do.  So the
state's relative error in the 2-norm is below 3 * 2 * 2^-16 < 2^-13, and o's below 2^-12 of its own and the largest
output, with half a step of its type on top."""
import numpy as np
import pytest
import torch

from conftest import announce, rel_l2
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STATE, OUT = 2.0 ** -13, 2.0 ** -12


class Case:
    """Inputs on the host and on the GPU; decays from 1 - 10^-3 to e^-3 a row."""

    def __init__(self, rows, hk, hv, slots, cuda, seed=0, gates=BF16, decay=1.0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.hk, self.hv = hk, hv
        self.y = torch.nn.functional.silu(r(rows, (2 * hk + hv) * 128)).to(BF16).to(cuda)
        self.a, self.b = (r(rows, hv).to(gates).to(cuda) for _ in range(2))
        self.A_log = torch.log(decay * (0.1 + 8 * torch.rand(hv, generator=g))).to(cuda)
        self.dt_bias = (r(hv) - 3).to(cuda)
        self.pool = (r(slots, hv, 128, 128) * 0.05).to(cuda)  # [slot, head, v, k]

    def check(self, cu=None, *, batch, limit, cu_host=None, indices=None, initial=None, o=None, o_dtype=None, scale=None,
              state=None, neg=False, label=""):
        from dforktree_amd import ops
        announce(f"prompt_gdn {label} rows={self.y.shape[0]} hk={self.hk} hv={self.hv} batch={batch} limit={limit}")
        state = self.pool.transpose(-1, -2) if state is None else state
        h = lambda t: t.double().cpu().numpy()  # noqa: E731
        rate = -torch.exp(self.A_log.float())
        want, want_state, want_status = P.prompt_gdn(
            h(self.y), h(self.a), h(self.b), h(rate), h(self.dt_bias), h(state), cu_host, hk=self.hk, hv=self.hv,
            batch=batch, limit=limit, scale=scale, indices=None if indices is None else indices.tolist(),
            initial=None if initial is None else initial.tolist())
        status = torch.full((batch,), -1, dtype=torch.int32, device=self.y.device)
        before = None if o is None else o.clone()
        old = state.clone()
        o = ops.prompt_gdn(self.y, self.a, self.b, None if neg else self.A_log, self.dt_bias, state, cu, hk=self.hk,
                           hv=self.hv, max_len=limit, batch=None if cu is not None else batch, scale=scale,
                           neg_exp_A=rate.contiguous() if neg else None, state_indices=indices, initial=initial, o=o,
                           o_dtype=o_dtype, status=status)
        assert status.tolist() == want_status.tolist()
        rows = ~np.isnan(want).any((1, 2))
        got = h(o)[rows]
        half = torch.finfo(o.dtype).eps / 2
        if rows.any():
            tol = half * np.abs(want[rows]) + OUT * (np.abs(want[rows]) + np.abs(want[rows]).max()) + (
                2.0 ** -25 if o.dtype == F16 else 0)
            assert (np.abs(got - want[rows]) <= tol).all(), (label, float(np.abs(got - want[rows]).max()))
        if before is not None:
            assert torch.equal(o[torch.tensor(~rows)], before[torch.tensor(~rows)])
        ws, gs = want_state, h(state)
        for s in range(state.shape[0]):
            if np.array_equal(ws[s], h(old[s])):
                assert torch.equal(state[s], old[s]), f"{label}: slot {s} was no request's"
            else:
                assert rel_l2(gs[s], ws[s]) <= STATE, (label, s, rel_l2(gs[s], ws[s]))
        return o


def cu_of(sizes, cuda):
    host = [0, *np.cumsum(sizes).tolist()]
    return host, torch.tensor(host, dtype=torch.int32, device=cuda)


def slots_of(B, n, cuda):
    return torch.randperm(n, generator=torch.Generator().manual_seed(B))[:B].to(cuda)


@pytest.mark.parametrize("sizes", [[1], [2], [16], [17], [63], [64], [65], [0, 1, 0, 3], [128, 1, 0, 129, 64],
                                   [200, 31, 97, 1, 1, 1], [1, 1, 1, 1, 300]])
@pytest.mark.parametrize("hk,hv", [(1, 1), (2, 4)])
def test_packed(cuda, sizes, hk, hv):
    host, cu = cu_of(sizes, cuda)
    B = len(sizes)
    c = Case(sum(sizes), hk, hv, B + 2, cuda, seed=len(sizes) + sum(sizes))
    init = torch.tensor([i % 3 != 1 for i in range(B)], device=cuda)
    c.check(cu, batch=B, limit=max(sizes), cu_host=host, indices=slots_of(B, B + 2, cuda), initial=init, label=str(sizes))


@pytest.mark.parametrize("sizes", [[1] * 200 + [300, 2, 16, 17, 15, 0, 64], [16] * 40 + [17] * 40, [5] * 140])
def test_many_requests_short_and_long(cuda, sizes):
    """From 512 heads on short requests go row by row beside long ones' chunks."""
    host, cu = cu_of(sizes, cuda)
    B = len(sizes)
    c = Case(sum(sizes), 2, 8, B + 2, cuda, seed=B)
    init = torch.tensor([i % 3 != 1 for i in range(B)], device=cuda)
    c.check(cu, batch=B, limit=max(sizes), cu_host=host, indices=slots_of(B, B + 2, cuda), initial=init, label="mixed")


def test_a_long_prompt(cuda):
    """Errors do not grow from chunk to chunk: 2500 rows, and states that keep them all."""
    for decay in (1e-3, 1.0):
        c = Case(2500, 1, 1, 1, cuda, seed=20, decay=decay)
        c.check(batch=1, limit=2500, o_dtype=F32, label=f"2500 rows, decay {decay}")


@pytest.mark.parametrize("hk,hv,batch", [(1, 1, 1), (1, 3, 2), (2, 8, 5), (16, 32, 3), (4, 4, 300)])
def test_tokens(cuda, hk, hv, batch):
    from dforktree_amd import ops
    c = Case(batch, hk, hv, batch + 1, cuda, seed=batch)
    at = slots_of(batch, batch + 1, cuda)
    pool = c.pool.clone()
    o = c.check(batch=batch, limit=1, indices=at, label="tokens")
    again = ops.token_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, pool.transpose(-1, -2), hk=hk, hv=hv, state_indices=at)
    assert torch.equal(o, again) and torch.equal(pool, c.pool)


@pytest.mark.parametrize("sizes", [[1, 1, 1], [70, 3]])
def test_padded_and_foreign_slots(cuda, sizes):
    """A negative slot starts from zeros and leaves nothing; so does one past the pool, with its status."""
    sizes = [*sizes, 5, 2]
    host, cu = cu_of(sizes, cuda)
    B = len(sizes)
    c = Case(sum(sizes), 1, 2, B, cuda, seed=1)
    at = torch.arange(B, device=cuda)
    at[0], at[-1] = -1, B
    c.check(cu, batch=B, limit=max(sizes), cu_host=host, indices=at.int(), label="slots")


@pytest.mark.parametrize("layout", ["k first", "k last", "odd rows", "odd base", "pitched"])
@pytest.mark.parametrize("sizes", [[1, 1], [100, 7]])
def test_state_layouts(cuda, layout, sizes):
    host, cu = cu_of(sizes, cuda)
    c = Case(sum(sizes), 1, 2, 3, cuda, seed=2)
    S = c.pool.transpose(-1, -2)  # [slot, head, k, v]
    if layout == "k first":
        state = S.contiguous()
    elif layout == "k last":
        state = S
    elif layout == "odd rows":
        state = torch.zeros(3, 2, 128, 129, device=cuda)[..., :128].transpose(-1, -2)
    elif layout == "odd base":
        state = torch.zeros(1 + c.pool.numel(), device=cuda)[1:].view(c.pool.shape).transpose(-1, -2)
    else:
        state = torch.zeros(3, 3, 130, 256, device=cuda)[:, 1:, :128, 64:192].transpose(-1, -2)
    state.copy_(S)
    c.check(cu, batch=2, limit=max(sizes), cu_host=host, state=state, label=layout)


@pytest.mark.parametrize("o_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("gates", [BF16, F16, F32])
def test_types(cuda, o_dtype, gates):
    host, cu = cu_of([90, 1, 40], cuda)
    c = Case(131, 1, 2, 3, cuda, seed=3, gates=gates)
    c.check(cu, batch=3, limit=90, cu_host=host, o_dtype=o_dtype, neg=gates == F32, scale=0.3, label=f"{o_dtype} {gates}")


def test_strides(cuda):
    """Rows of a wider projection (16-byte aligned or not), gates as columns of one, outputs within a wider buffer."""
    host, cu = cu_of([70, 1, 20], cuda)
    for shift in (8, 3):
        c = Case(91, 1, 2, 3, cuda, seed=4)
        wide = torch.randn(91, 544, device=cuda).bfloat16()
        wide[:, shift:shift + 512] = c.y
        c.y = wide[:, shift:shift + 512]
        ab = torch.stack([c.a, c.b], 1).view(91, 4)
        c.a, c.b = ab[:, :2], ab[:, 2:]
        out = torch.zeros(91, 3, 131, device=cuda).bfloat16()
        c.check(cu, batch=3, limit=70, cu_host=host, o=out[:, 1:, 2:130], label=f"shift {shift}")
        assert not out[:, 0].any() and not out[:, :, :2].any() and not out[:, :, 130:].any()


@pytest.mark.parametrize("limit", [1, 30, 64])
def test_cut_requests(cuda, limit):
    for host in ([3, 60, 61, 120, 170], [0, 90, 80, 90, 130]):
        c = Case(130, 1, 2, 4, cuda, seed=5)
        out = torch.full((130, 2, 128), 3.0, dtype=BF16, device=cuda)
        cu = torch.tensor(host, dtype=torch.int32, device=cuda)
        c.check(cu, batch=4, limit=limit, cu_host=host, o=out, label=f"{host} {limit}")


@pytest.mark.parametrize("decay", [1e-4, 1.0, 30.0, 1000.0])
@pytest.mark.parametrize("n", [1, 130])
def test_decays(cuda, decay, n):
    """From almost none to ones that leave nothing of a row after the next."""
    c = Case(n, 1, 2, 1, cuda, seed=6, decay=decay)
    c.check(batch=1, limit=n, label=f"decay {decay}")


@pytest.mark.parametrize("kind", ["write all", "write none", "zero rows", "same keys", "large values", "gate 20"])
@pytest.mark.parametrize("n", [1, 150])
def test_extremes(cuda, kind, n):
    c = Case(n, 1, 2, 1, cuda, seed=7)
    if kind == "write all":
        c.b.fill_(100)
    elif kind == "write none":
        c.b.fill_(-100)
    elif kind == "zero rows":
        c.y[::3] = 0
    elif kind == "same keys":  # the largest A: every key the same, all of it written
        c.y[:, 128:256] = c.y[0, 128:256].clone()
        c.b.fill_(100)
        c.A_log.fill_(-9)
    elif kind == "large values":
        c.y[:, 256:] *= 1000
    else:
        c.a.copy_(torch.linspace(18, 26, 2 * n).view(n, 2))
        c.dt_bias.zero_()
        c.A_log.fill_(-6)
    c.check(batch=1, limit=n, label=kind)


@pytest.mark.parametrize("sizes", [[1, 1], [70, 65]])
def test_not_finite_elsewhere(cuda, sizes):
    """Rows of no request, and slots that nobody goes on from, are not read; a request that is not finite keeps it."""
    host, cu = cu_of(sizes, cuda)
    c = Case(sum(sizes) + 40, 1, 2, 3, cuda, seed=8)
    for t in (c.y, c.a, c.b):
        t[sum(sizes):] = float("nan")
    c.pool[1] = float("nan")
    c.pool[2] = float("inf")
    init = torch.tensor([True, False], device=cuda)
    out = torch.zeros(c.y.shape[0], 2, 128, dtype=BF16, device=cuda)
    c.pool[2] = 0  # (the oracle compares slots)
    c.check(cu, batch=2, limit=max(sizes), cu_host=host, initial=init, o=out, label="not finite")
    # a NaN in the last row of the first request touches neither its earlier chunks nor the second request
    from dforktree_amd import ops
    c = Case(sum(sizes), 1, 2, 2, cuda, seed=9)
    args = lambda s: (c.y, c.a, c.b, c.A_log, c.dt_bias, s.transpose(-1, -2), cu)  # noqa: E731
    clean, kept = c.pool.clone(), c.pool.clone()
    o = ops.prompt_gdn(*args(clean), hk=1, hv=2, max_len=max(sizes))
    c.y[sizes[0] - 1] = float("nan")
    spoiled = ops.prompt_gdn(*args(kept), hk=1, hv=2, max_len=max(sizes))
    first = (sizes[0] - 1) // 64 * 64
    assert torch.equal(spoiled[:first], o[:first]) and torch.equal(spoiled[sizes[0]:], o[sizes[0]:])
    assert torch.equal(kept[1], clean[1]) and kept[0].isnan().any() and spoiled[sizes[0] - 1].isnan().any()


def test_in_pieces(cuda):
    """A prompt in chunks of any length leaves what the whole leaves, within both runs' tolerances."""
    from dforktree_amd import ops
    announce("prompt_gdn in pieces")
    c = Case(333, 2, 4, 1, cuda, seed=10)
    whole, part = c.pool.clone(), c.pool.clone()
    run = lambda s, i, j: ops.prompt_gdn(c.y[i:j], c.a[i:j], c.b[i:j], c.A_log, c.dt_bias, s.transpose(-1, -2),  # noqa: E731
                                         hk=2, hv=4, o_dtype=F32)
    o = run(whole, 0, 333)
    cuts = [0, 1, 2, 66, 130, 131, 333]
    parts = torch.cat([run(part, i, j) for i, j in zip(cuts, cuts[1:])])
    assert rel_l2(part.cpu(), whole.cpu()) <= 2 * STATE and rel_l2(parts.cpu(), o.cpu()) <= 2 * OUT


def test_a_chain_of_tree_nodes(cuda):
    """A chain verified as a tree and committed is the same rows as a prompt's chunk."""
    from dforktree_amd import ops
    announce("prompt_gdn against tree_verify and tree_commit")
    n, hk, hv = 16, 2, 4
    c = Case(n, hk, hv, 1, cuda, seed=11)
    ts = ops.tree_struct(torch.arange(-1, n - 1, device=cuda), 4, batch=1, n_nodes=n, want=("anc_bits",))
    k, v, g = (torch.zeros(1, hv, n, *d, device=cuda) for d in ((128,), (128,), ()))
    tree = c.pool.clone()
    o = ops.tree_verify(c.y, c.a, c.b, c.A_log, c.dt_bias, tree.transpose(-1, -2), hk=hk, hv=hv, anc_bits=ts["anc_bits"],
                        aux_k=k[0], aux_v=v[0], aux_g=g[0], o_dtype=F32)
    ops.tree_commit(tree.unsqueeze(0), k, v, g, torch.arange(n, device=cuda)[None], n_nodes=n)
    mine = ops.prompt_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, c.pool.transpose(-1, -2), hk=hk, hv=hv, o_dtype=F32)
    assert rel_l2(mine.cpu(), o.cpu()) <= 2 * OUT and rel_l2(c.pool.cpu(), tree.cpu()) <= 2 * STATE


@pytest.mark.parametrize("n", [1, 70])
def test_offsets_past_32_bits(cuda, n):
    """Rows 2^25 elements apart, a slot past 2^31 elements of the pool."""
    from dforktree_amd import ops
    announce(f"prompt_gdn offsets past 32 bits n={n}")
    c = Case(n, 1, 2, 1, cuda, seed=12)
    y = torch.empty(n << 25, dtype=BF16, device=cuda).as_strided(c.y.shape, (1 << 25, 1)).copy_(c.y)
    o = torch.empty(n << 25, dtype=BF16, device=cuda).as_strided((n, 2, 128), (1 << 25, 128, 1))
    pool = torch.empty((1 << 31) + 2 * 16384, device=cuda).as_strided((2, 2, 128, 128), (1 << 31, 16384, 128, 1))
    pool.copy_(c.pool.expand(2, -1, -1, -1))
    gates = (c.a, c.b, c.A_log, c.dt_bias)
    ops.prompt_gdn(y, *gates, pool.transpose(-1, -2), hk=1, hv=2, state_indices=torch.tensor([1], device=cuda), o=o)
    near = c.pool.clone()
    assert torch.equal(o, ops.prompt_gdn(c.y, *gates, near.transpose(-1, -2), hk=1, hv=2))
    assert torch.equal(pool[1], near[0]) and torch.equal(pool[0], c.pool[0])


@pytest.mark.parametrize("sizes", [[1] * 5, [100, 64, 1]])
def test_captured_and_on_another_stream(cuda, sizes):
    """Replays go on from where the last one ended, with the lengths that its buffers hold; two graphs side by side do not
    share a workspace."""
    from dforktree_amd import ops
    announce(f"prompt_gdn in a graph {sizes}")
    host, cu = cu_of(sizes, cuda)
    B, T = len(sizes), sum(sizes)
    c, d = (Case(T, 1, 2, B, cuda, seed=s) for s in (13, 14))
    eager = c.pool.clone(), d.pool.clone()
    kw = dict(hk=1, hv=2, max_len=max(sizes))
    run = lambda c, pool, o=None: ops.prompt_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, pool.transpose(-1, -2), cu, o=o, **kw)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = run(c, c.pool.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in (c, d):
        graphs.append(torch.cuda.CUDAGraph())
        outs.append(torch.empty_like(warm))
        with torch.cuda.graph(graphs[-1]):
            run(x, x.pool, outs[-1])
    assert torch.equal(warm, run(c, eager[0].clone()))
    for step in range(4):
        for x in (c, d):
            x.y.copy_(torch.randn(x.y.shape, generator=torch.Generator().manual_seed(step)))
        if step == 2:  # other lengths in the same buffers
            cu.copy_(torch.tensor([0, *np.cumsum(sizes[::-1]).tolist()], dtype=torch.int32))
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for x, e, o in zip((c, d), eager, outs):
            assert torch.equal(o, run(x, e)) and torch.equal(x.pool, e)
        torch.cuda.synchronize()


def test_two_at_once(cuda):
    """Two calls on streams of their own, each with chunks and its own workspace."""
    from dforktree_amd import ops
    announce("prompt_gdn on two streams")
    cases = [Case(200, 2, 4, 3, cuda, seed=s) for s in (31, 32)]
    cu = torch.tensor([0, 70, 71, 200], dtype=torch.int32, device=cuda)
    run = lambda c, pool: ops.prompt_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, pool.transpose(-1, -2), cu, hk=2, hv=4,  # noqa: E731
                                         max_len=129)
    want = []
    for c in cases:
        pool = c.pool.clone()
        want.append((run(c, pool), pool))
    pools = [[c.pool.clone() for _ in range(6)] for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for i in range(6):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(run(cases[k], pools[k][i]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for o, pool in zip(got[k], pools[k]):
            assert torch.equal(o, want[k][0]) and torch.equal(pool, want[k][1])


def test_same_on_every_run(cuda):
    """No sum depends on the order in which workgroups finish, or on the requests beside one."""
    from dforktree_amd import ops
    announce("prompt_gdn runs alike")
    sizes = [200, 1, 65, 64]
    host, cu = cu_of(sizes, cuda)
    c = Case(sum(sizes), 2, 4, 4, cuda, seed=15)
    pools = [c.pool.clone() for _ in range(3)]
    run = lambda p, **kw: ops.prompt_gdn(c.y, c.a, c.b, c.A_log, c.dt_bias, p.transpose(-1, -2), cu, hk=2, hv=4,  # noqa: E731
                                         max_len=200, **kw)
    o = [run(p) for p in pools]
    assert all(torch.equal(o[0], x) for x in o) and all(torch.equal(pools[0], p) for p in pools)


def test_refused(cuda):
    from dforktree_amd import ops
    c = Case(6, 1, 2, 2, cuda)
    S = c.pool.transpose(-1, -2)
    base = dict(y=c.y, a=c.a, b=c.b, A_log=c.A_log, dt_bias=c.dt_bias, state=S, hk=1, hv=2)
    for kw, err in ((dict(y=c.y.float()), TypeError), (dict(y=c.y[:, :500]), ValueError), (dict(y=c.y[0]), ValueError),
                    (dict(a=c.a[:, :1]), ValueError), (dict(b=c.b[:3]), ValueError), (dict(A_log=None), ValueError),
                    (dict(dt_bias=c.dt_bias[:1]), ValueError), (dict(neg_exp_A=c.A_log.half()), TypeError),
                    (dict(state=S.half()), TypeError), (dict(state=S[0]), ValueError), (dict(state=S[:, :1]), ValueError),
                    (dict(state=S[:1].expand(2, -1, -1, -1)), ValueError), (dict(hk=0), ValueError),
                    (dict(hk=3, hv=4), ValueError), (dict(max_len=4, batch=2), ValueError),
                    (dict(state_indices=torch.zeros(2, dtype=torch.int32, device=cuda)), ValueError),
                    (dict(initial=torch.zeros(1, device=cuda)), TypeError), (dict(a=c.a.int()), TypeError),
                    (dict(o=torch.empty(6, 2, 64, device=cuda)), ValueError), (dict(o_dtype=torch.int32), TypeError),
                    (dict(cu_seqlens=torch.tensor([0, 6], dtype=torch.int32, device=cuda)), ValueError),
                    (dict(state=S.cpu()), ValueError), (dict(max_len=2, batch=3), ValueError)):
        with pytest.raises(err):
            ops.prompt_gdn(**(base | kw))
    with pytest.raises(ValueError):
        ops.token_gdn(**base)  # 6 tokens, 2 slots
    assert ops.prompt_gdn(**(base | dict(y=c.y[:0], a=c.a[:0], b=c.b[:0], max_len=0, batch=2))).shape == (0, 2, 128)
