"""ops.tree_accept against the 64-bit oracle: whole numbers, equal."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def tree(n, kind, rng):
    if kind == "chain":
        return [-1, *range(n - 1)][:n]
    if kind == "star":
        return ([-1] + [0] * n)[:n]
    return ([-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)])[:n]


class Case:
    def __init__(self, sizes, V, kind, drawn, seed, *, dtype=F32, index=torch.int32, sharp=2.0, cu=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.cu = [0, *np.cumsum(sizes).tolist()] if cu is None else cu
        T = sum(sizes)
        parents = [tree(n, kind, rng) for n in sizes]
        self.parent = torch.tensor(sum(parents, []), dtype=index)
        logits = sharp * torch.randn(T, V, generator=g)
        self.probs = torch.softmax(logits, 1).to(dtype)
        other = logits + 0.5 * torch.randn(T, V, generator=g)
        self.draft = torch.softmax(other, 1).to(dtype) if drawn else None
        order = torch.argsort(other, 1, descending=True)
        tokens, row = [], 0
        for p in parents:  # the likeliest tokens, so that some stand
            for i in range(len(p)):
                place = p[1:i].count(p[i]) if i else 0
                tokens.append(int(order[row + max(p[i], 0), place % V]))
            row += len(p)
        self.tokens = torch.tensor(tokens, dtype=index)
        self.u, self.last = torch.rand(T, generator=g), torch.rand(len(sizes), generator=g)

    def check(self, cuda, *, cols=16, limit=None, uniform=False, label=""):
        from dforktree_amd import ops
        B, T = len(self.last), len(self.tokens)
        limit = max(b - a for a, b in zip(self.cu, self.cu[1:])) if limit is None else limit
        announce(f"tree_accept {label} B={B} T={T} V={self.probs.shape[1]} {self.probs.dtype} cols={cols} limit={limit}")
        d = lambda t: None if t is None else t.to(cuda) if t.device != cuda else t  # noqa: E731
        status = torch.full((B,), -1, dtype=torch.int32, device=cuda)
        kw = dict(batch=B) if uniform else dict(cu_seqlens=torch.tensor(self.cu, dtype=torch.int32, device=cuda))
        got = ops.tree_accept(d(self.tokens), d(self.parent), d(self.probs), d(self.u), d(self.last),
                              draft_probs=d(self.draft), n_nodes=limit, path_cols=cols, status=status, **kw)
        path, rows = np.full((B, cols), -1), np.full((B, cols), -1)
        length, token, want = np.zeros(B, int), np.zeros(B, int), np.zeros(B, int)
        h = lambda t: t.double().cpu().numpy()  # noqa: E731
        for b, (r0, n, st) in enumerate(P.spans(None if uniform else self.cu, B, limit, T)):
            r = slice(r0, r0 + n)
            p, token[b] = P.accept(self.tokens[r].tolist(), self.parent[r].tolist(), h(self.probs[r]), h(self.u[r]),
                                   float(self.last[b]), None if self.draft is None else h(self.draft[r]), cols)
            length[b], path[b, :len(p)], rows[b, :len(p)] = len(p), p, [r0 + x for x in p]
            want[b] = st | (P.STATUS_WEIGHT if n and token[b] < 0 else 0)
        assert got["path"].tolist() == path.tolist(), label
        assert got["path_len"].tolist() == length.tolist() and got["rows"].tolist() == rows.tolist()
        assert got["token"].tolist() == token.tolist(), label
        assert status.tolist() == want.tolist()
        return got


@pytest.mark.parametrize("V", [1, 2, 5, 63, 1000, 1025, 4099, 20001])
@pytest.mark.parametrize("kind", ["chain", "tree", "star"])
@pytest.mark.parametrize("drawn", [False, True])
def test_trees(cuda, V, kind, drawn):
    c = Case([1, 5, 0, 16, 33, 2, 64], V, kind, drawn, seed=V)
    got = c.check(cuda, label=f"{kind} drawn={drawn}")
    if V == 63 and kind == "tree":
        assert got["path_len"].max() > 2  # the cases reach further than the root


@pytest.mark.parametrize("seed", range(6))
def test_many_refusals(cuda, seed):
    """Stars whose every child may fall: up to 63 reductions of one row, and repeated tokens where V is small."""
    for V in (40, 300):
        c = Case([64, 20, 64, 40], V, "star", True, seed, sharp=0.5)
        c.u.fill_(1 - 2.0 ** -24)  # refused unless the target has at least the drafter's share
        c.check(cuda, label="refused")
        c.draft = None
        c.check(cuda, label="refused, not drawn")


@pytest.mark.parametrize("V", [131072, 100003])
@pytest.mark.parametrize("drawn", [False, True])
def test_large_vocabulary(cuda, V, drawn):
    c = Case([9, 1, 12], V, "tree", drawn, seed=1)
    for last in (0.0, 0.25, 1 - 2.0 ** -24):
        c.last.fill_(last)
        c.check(cuda, label=f"last={last}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("drawn", [False, True])
def test_types(cuda, dtype, index, drawn):
    Case([7, 12, 30], 777, "tree", drawn, seed=2, dtype=dtype, index=index).check(cuda, label=f"{dtype} {index}")


@pytest.mark.parametrize("cols", [1, 2, 5, 64])
def test_path_columns(cuda, cols):
    for kind in ("chain", "tree"):
        for drawn in (False, True):
            c = Case([40, 64, 3], 6, kind, drawn, seed=3)
            c.u.mul_(0.2)  # long paths
            c.check(cuda, cols=cols, label=f"cols {kind}")


def test_every_node_stands(cuda):
    for drawn in (False, True):
        c = Case([64, 64], 50, "chain", drawn, seed=4)
        c.u.zero_()
        got = c.check(cuda, cols=64, label="all stand")
        assert got["path_len"].tolist() == [64, 64]


def test_drafter_is_the_target(cuda):
    """Whatever is drawn from the target's own distribution stands."""
    c = Case([20, 9], 500, "chain", True, seed=5)
    c.draft = c.probs.clone()
    assert c.check(cuda, cols=32, label="the same")["path_len"].tolist() == [20, 9]


def test_sharp_rows(cuda):
    """Rows with one token of weight, in the target's, the drafter's or both."""
    for drawn in (False, True):
        c = Case([30, 31, 32], 9, "tree", drawn, seed=6)
        for rows, p in ((slice(0, 60), c.probs), (slice(20, 93), c.draft)):
            if p is not None:
                p[rows] = 0
                p[rows, 4] = 1
        c.check(cuda, label="one-hot")
        c.tokens.fill_(4)
        c.check(cuda, label="one-hot, all of one token")


@pytest.mark.parametrize("drawn", [False, True])
def test_without_weight_and_strange_values(cuda, drawn):
    c = Case([10, 10, 10, 10, 10], 130, "tree", drawn, seed=7)
    c.probs[:10] = 0
    c.probs[10:20] = float("nan")
    c.probs[20:30, ::2] = -0.5
    c.probs[30:40, 100:] = float("nan")
    if drawn:
        c.draft[20:30, 1::2] = 0
        c.draft[40:50, ::3] = float("nan")
    c.check(cuda, label="strange values")


@pytest.mark.parametrize("drawn", [False, True])
def test_tokens_outside_the_vocabulary(cuda, drawn):
    c = Case([20, 20, 20], 40, "tree", drawn, seed=8, index=torch.int64)
    c.tokens[1::4] = -1
    c.tokens[2::4] = 40
    c.tokens[5] = 1 << 40
    c.tokens[0::20] = -7  # a root's is not read
    c.check(cuda, label="outside")


def test_strange_parents(cuda):
    """A negative parent is the root; a node whose parent is not in front of it is never reached."""
    c = Case([12, 12], 6, "tree", False, seed=9)
    c.u.mul_(0.3)
    c.parent[3], c.parent[5], c.parent[14], c.parent[16] = -5, 5, 9, 100
    c.check(cuda, label="parents")


@pytest.mark.parametrize("drawn", [False, True])
def test_cut_requests(cuda, drawn):
    c = Case([30, 30, 30], 50, "tree", drawn, seed=10, cu=[4, 30, 61, 95])
    c.check(cuda, limit=20, label="cut")
    c.cu = [0, 40, 30, 90]
    c.check(cuda, limit=64, label="not in order")


@pytest.mark.parametrize("n", [1, 16])
def test_uniform_rows(cuda, n):
    c = Case([n] * 5, 100, "tree", True, seed=11)
    c.check(cuda, limit=n, uniform=True, label="uniform")


def test_strides(cuda):
    """Rows of a wider buffer, at addresses of any alignment."""
    for drawn in (False, True):
        c = Case([9, 30, 4], 1001, "tree", drawn, seed=12)
        for name in ("probs", "draft"):
            t = getattr(c, name)
            if t is not None:
                wide = torch.full((43, 1303), float("nan"), device=cuda)
                wide[:, 7:1008] = t
                setattr(c, name, wide[:, 7:1008])
        c.check(cuda, label="strided")


@pytest.mark.parametrize("V", [3, 1001, 20000])
def test_rows_of_unlike_alignment(cuda, V):
    """The drafter's rows start elsewhere in a piece of four than the target's."""
    c = Case([9, 30, 4], V, "star", True, seed=16)
    c.u.fill_(1 - 2.0 ** -24)
    for name, at, width in (("probs", 3, V + 6), ("draft", 5, V + 9)):
        wide = torch.full((43, width), float("nan"), device=cuda)
        wide[:, at:at + V] = getattr(c, name)
        setattr(c, name, wide[:, at:at + V])
    c.check(cuda, label="unlike alignment")


@pytest.mark.parametrize("seed", range(3))
def test_many_refusals_over_long_rows(cuda, seed):
    """More passes over whole rows than launches make, beside requests of few."""
    c = Case([40, 3, 64, 1, 9], 20001 + seed, "star" if seed else "tree", True, seed=40 + seed, sharp=0.3)
    c.u.fill_(1 - 2.0 ** -24)
    c.check(cuda, label="refused over long rows")


def test_captured_over_long_rows(cuda):
    from dforktree_amd import ops
    announce("tree_accept over long rows in a graph")
    c = Case([30, 9, 20], 30001, "tree", True, seed=19)
    t = [x.to(cuda) for x in (c.tokens, c.parent, c.probs, c.u, c.last, c.draft)]
    cu = torch.tensor(c.cu, dtype=torch.int32, device=cuda)
    run = lambda: ops.tree_accept(*t[:5], draft_probs=t[5], cu_seqlens=cu, n_nodes=30)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(4):
        g = torch.Generator().manual_seed(step)
        t[3].copy_(torch.rand(59, generator=g) ** (0.2 if step % 2 else 1))
        t[4].copy_(torch.rand(3, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        for k in out:
            assert torch.equal(out[k], want[k]), (step, k)


def test_no_vocabulary(cuda):
    from dforktree_amd import ops
    announce("tree_accept without tokens")
    i, p, u = torch.zeros(5, dtype=torch.int32, device=cuda), torch.ones(5, 0, device=cuda), torch.rand(5, device=cuda)
    for draft in (None, p):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        got = ops.tree_accept(i, i, p, u, u[:1], draft_probs=draft, status=status)
        assert got["token"].tolist() == [-1] and got["path_len"].tolist() == [1]
        assert got["path"][0].tolist() == [0] + [-1] * 15 and status.tolist() == [P.STATUS_WEIGHT]


def test_two_at_once(cuda):
    """Two calls on streams of their own."""
    from dforktree_amd import ops
    announce("tree_accept on two streams")
    cases = [Case([33, 64, 20], 20001, "tree", True, seed=s) for s in (17, 18)]
    args = [([x.to(cuda) for x in (c.tokens, c.parent, c.probs, c.u, c.last)],
             dict(draft_probs=c.draft.to(cuda), cu_seqlens=torch.tensor(c.cu, dtype=torch.int32, device=cuda), n_nodes=64))
            for c in cases]
    want = [ops.tree_accept(*t, **kw) for t, kw in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.tree_accept(*args[k][0], **args[k][1]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for g in got[k]:
            assert all(torch.equal(g[n], want[k][n]) for n in g)


def test_offsets_past_32_bits(cuda):
    c = Case([9, 30, 4], 1001, "tree", True, seed=13)
    for name in ("probs", "draft"):
        far = torch.empty(43 << 26, dtype=BF16, device=cuda).as_strided((43, 1001), (1 << 26, 1))
        setattr(c, name, far.copy_(getattr(c, name)))
    c.check(cuda, label="far rows")


def test_many_requests(cuda):
    sizes = [1 + i % 9 for i in range(700)]
    for drawn in (False, True):
        Case(sizes, 60, "tree", drawn, seed=14).check(cuda, label="700 requests")


def test_captured(cuda):
    """A captured step takes new numbers, probabilities and lengths; every replay is the eager result."""
    from dforktree_amd import ops
    announce("tree_accept in a graph")
    c = Case([16, 9, 20], 3001, "tree", True, seed=15)
    cu = torch.tensor(c.cu, dtype=torch.int32, device=cuda)
    t = [x.to(cuda) for x in (c.tokens, c.parent, c.probs, c.u, c.last, c.draft)]
    run = lambda: ops.tree_accept(*t[:5], draft_probs=t[5], cu_seqlens=cu, n_nodes=20)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(4):
        g = torch.Generator().manual_seed(step)
        t[3].copy_(torch.rand(45, generator=g))
        t[4].copy_(torch.rand(3, generator=g))
        t[2].copy_(t[2].roll(1, 0))
        if step == 2:
            cu.copy_(torch.tensor([0, 9, 25, 45]))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        for k in out:
            assert torch.equal(out[k], want[k]), (step, k)


def test_refused(cuda):
    from dforktree_amd import ops
    i, p, u = torch.zeros(6, dtype=torch.int32, device=cuda), torch.ones(6, 9, device=cuda), torch.rand(6, device=cuda)
    base = dict(tokens=i, parent=i, probs=p, uniform=u, last=u[:1])
    for kw, err in ((dict(tokens=u), TypeError), (dict(parent=i[:3]), ValueError), (dict(probs=p[:3]), ValueError),
                    (dict(probs=p[0]), ValueError), (dict(probs=p.int()), TypeError),
                    (dict(probs=torch.ones(9, 6, device=cuda).t()), ValueError), (dict(draft_probs=p[:, :4]), ValueError),
                    (dict(draft_probs=p.int()), TypeError), (dict(uniform=u[:2]), ValueError),
                    (dict(uniform=u.double()), TypeError), (dict(last=u[:2]), ValueError),
                    (dict(last=u[:1].half()), TypeError), (dict(path_cols=0), ValueError), (dict(path_cols=65), ValueError),
                    (dict(n_nodes=4, batch=2), ValueError), (dict(probs=p.cpu()), ValueError),
                    (dict(cu_seqlens=torch.tensor([0, 6], device=cuda)), TypeError)):
        with pytest.raises(err):
            ops.tree_accept(**(base | kw))
    n = 65
    i, p, u = torch.zeros(n, dtype=torch.int32, device=cuda), torch.ones(n, 9, device=cuda), torch.rand(n, device=cuda)
    with pytest.raises(ValueError, match="64"):
        ops.tree_accept(i, i, p, u, u[:1])
    e = ops.tree_accept(i[:0], i[:0], p[:0], u[:0], u[:2], n_nodes=0, batch=2)
    assert e["path_len"].tolist() == [0, 0] and e["token"].tolist() == [-1, -1] and (e["path"] == -1).all()
