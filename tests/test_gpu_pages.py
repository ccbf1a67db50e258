"""Page plans and cache writes: whole numbers and copies, equal bit for bit."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P

pytestmark = pytest.mark.gpu


def tables(rng, held, cols, extra):
    pages = int(sum(held)) + extra
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(held), cols), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table, order[at:]


def compare(cuda, prefix, new, table, held, ring, pos, *, ps, rows, trim=False, depth=None, index=torch.int32, times=2,
            stride=0, **kw):
    from dforktree_amd import ops
    want = P.page_plan(prefix, new, table, held, ring, pos, page_size=ps, rows=rows, trim=trim, depth=depth)
    ints = lambda x, dt=torch.int32: torch.tensor(np.asarray(x), dtype=dt, device=cuda)  # noqa: E731
    cols = table.shape[1]
    wide = torch.full((len(held), cols + stride), -9, dtype=torch.int32, device=cuda)
    t = wide[:, :cols]
    t.copy_(ints(table))
    r, p = ints(ring), ints(pos, torch.int64)
    for _ in range(times):  # the second call finds what the first wrote
        got = ops.page_plan(ints(prefix, index), ints(new, index), t, ints(held), r, p, page_size=ps, rows=rows, trim=trim,
                            depth=None if depth is None else ints(depth, index), **kw)
        torch.cuda.synchronize()
        for name in ("status", "cu_seqlens", "held", "free_pos", "seq_len", "slots", "positions"):
            assert np.array_equal(got[name].cpu().numpy(), want[name]), name
        assert np.array_equal(t.cpu().numpy(), want["block_table"]) and (wide[:, cols:] == -9).all()
        assert np.array_equal(r.cpu().numpy(), want["free_pages"])
        assert p.tolist() == list(pos)
    return want


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 255, 257, 1000])
@pytest.mark.parametrize("ps", [1, 16, 24])
@pytest.mark.parametrize("trim", [False, True])
def test_random_plans(cuda, batch, ps, trim):
    announce(f"plan batch={batch} ps={ps} trim={trim}")
    rng = np.random.default_rng(batch * 100 + ps)
    prefix, new = rng.integers(0, 300, batch), rng.integers(0, 40, batch)
    new[rng.random(batch) < 0.2] = 0
    held = -(-prefix // ps) + rng.integers(0, 4, batch) * (rng.random(batch) < 0.5)
    held[rng.random(batch) < 0.1] = 0
    cols = 360 // ps + 6
    table, free = tables(rng, held, cols, 340 * batch // ps + 3)
    head = int(rng.integers(0, 1 << 40))
    cap = int(sum(held)) + len(free)
    ring = np.full(cap, -1, np.int32)
    ring[(head + np.arange(len(free))) % cap] = free
    rows = int(new.sum())
    compare(cuda, prefix, new, table, held, ring, [head, head + len(free)], ps=ps, rows=rows, trim=trim,
            index=torch.int64 if batch % 2 else torch.int32, stride=batch % 3)


def test_plans_that_do_not_fit(cuda):
    """Too few pages, too few columns, too few rows, no room in the ring, negative and empty."""
    announce("plans that do not fit")
    rng = np.random.default_rng(1)
    prefix, new = np.array([10, 0, 200, -4, 7, 50, 0]), np.array([20, 33, 9, 5, -3, 1, 64])
    held = np.array([1, 0, 13, 0, 1, 4, 0])
    for free, rows, cap in ((0, 132, 60), (2, 132, 60), (3, 40, 60), (9, 132, 30), (60, 3, 60), (40, 0, 41)):
        table, pages = tables(rng, held, 14, 60)
        ring = np.full(cap, -1, np.int32)
        k = min(free, cap)
        ring[(5 + np.arange(k)) % cap] = pages[:k]
        for trim in (False, True):
            want = compare(cuda, prefix, new, table, held, ring, [5, 5 + k], ps=16, rows=rows, trim=trim)
            assert want["status"][3] & P.STATUS_SPAN
    table, pages = tables(rng, [3, 0], 2 + 1, 9)
    want = compare(cuda, [0, 0], [0, 100], table, [3, 0], pages[:9], [0, 9], ps=16, rows=120, trim=True)
    assert want["status"].tolist() == [P.STATUS_PAGES, P.STATUS_TABLE]  # a full ring; a table of three columns
    compare(cuda, [], [], np.zeros((0, 3), np.int32), [], pages, [2, 5], ps=4, rows=5)
    compare(cuda, [4], [0], np.full((1, 2), 7, np.int32), [1], pages, [2, 5], ps=4, rows=0)


def test_tree_positions_and_long_rows(cuda):
    announce("tree positions")
    rng = np.random.default_rng(3)
    new = rng.integers(1, 65, 70)
    prefix = rng.integers(0, 5000, 70)
    held = -(-prefix // 1)
    table, free = tables(rng, held, 5070, 5000)
    compare(cuda, prefix, new, table, held, free, [0, len(free)], ps=1, rows=int(new.sum()) + 9,
            depth=rng.integers(0, 20, int(new.sum()) + 9), times=1)
    table, free = tables(rng, [0, 3], 20000, 20003)  # a whole prompt at one token a page
    compare(cuda, [0, 3], [20000, 1], table, [0, 3], free, [7, 7 + len(free)], ps=1, rows=20001, times=1)


def test_index_types_and_graph(cuda):
    from dforktree_amd import ops
    announce("plan graph")
    ints = lambda x, dt=torch.int32: torch.tensor(x, dtype=dt, device=cuda)  # noqa: E731
    prefix, new, held = ints([3, 20]), ints([1, 1]), ints([1, 2])
    table = ints([[4, -1, -1], [5, 6, -1]])
    ring, pos = ints([7, 8, 9, 10, -1, -1, -1]), ints([0, 4], torch.int64)
    call = lambda: ops.page_plan(prefix, new, table, held, ring, pos, page_size=16, rows=2, index_dtype=torch.int32)  # noqa: E731
    r = call()
    assert r["slots"].dtype == r["positions"].dtype == torch.int32 and r["slots"].tolist() == [67, 100]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = call()
    for p in ([3, 20], [16, 31], [15, 32], [3, 20]):
        prefix.copy_(ints(p))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = P.page_plan(p, [1, 1], [[4, -1, -1], [5, 6, -1]], [1, 2], [7, 8, 9, 10, -1, -1, -1], [0, 4], page_size=16, rows=2)
        assert r["slots"].tolist() == want["slots"].tolist() and r["free_pos"].tolist() == want["free_pos"].tolist()


@pytest.mark.parametrize("heads,d", [(1, 64), (2, 128), (8, 128), (3, 256), (2, 36), (5, 7)])
@pytest.mark.parametrize("src,dst", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "bfloat16"),
                                     ("bfloat16", "float16"), ("float32", "float32")])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append(cuda, heads, d, src, dst, heads_first):
    from dforktree_amd import ops
    announce(f"append {heads}x{d} {src}->{dst} heads_first={heads_first}")
    src, dst = getattr(torch, src), getattr(torch, dst)
    g = torch.Generator().manual_seed(heads * d)
    for n, pages, ps in ((1, 1, 1), (37, 9, 5), (300, 21, 16)):
        kv = torch.randn(n, 2, heads, d, generator=g).to(src)
        shape = (pages, heads, ps, d) if heads_first else (pages, ps, heads, d)
        caches = [torch.randn(shape, generator=g).to(dst) for _ in range(2)]
        slots = torch.randperm(pages * ps, generator=g)[:min(n, pages * ps)]
        m = len(slots)
        slots[torch.rand(m, generator=g) < 0.1] = -1
        view = lambda c: c.transpose(1, 2) if heads_first else c  # noqa: E731
        wk, wv, _ = P.kv_append(kv[:, 0].to(dst).float().numpy(), kv[:, 1].to(dst).float().numpy(),
                                view(caches[0]).float().numpy(), view(caches[1]).float().numpy(), slots.tolist())
        x = kv.to(cuda)
        kc, vc = (view(c.to(cuda)) for c in caches)
        ops.kv_append(x[:, 0], x[:, 1], kc, vc, slots.to(cuda, torch.int32 if n == 37 else torch.int64))
        torch.cuda.synchronize()
        assert np.array_equal(kc.float().cpu().numpy(), wk) and np.array_equal(vc.float().cpu().numpy(), wv)


def test_append_of_paths_and_bad_entries(cuda):
    """A row gather with gaps; slots and rows past the ends are skipped and marked; bits survive (NaN, -0)."""
    from dforktree_amd import ops
    announce("append paths")
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(64, 2, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    k[3, 0, 0], k[3, 0, 1], v[3, 1, 2] = float("nan"), -0.0, float("inf")
    rows = torch.tensor([0, 3, -1, 63, 64, 5, 2, -2])
    slots = torch.tensor([7, 0, 1, 47, 3, 48, -1, 9])
    for entries, word in ((8, 1), (4, 0)):
        kc, vc = (torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16, device=cuda) for _ in range(2))
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        ops.kv_append(k.to(cuda), v.to(cuda), kc, vc, slots[:entries].to(cuda), rows=rows[:entries].to(cuda), status=status)
        torch.cuda.synchronize()
        wk, wv, _ = P.kv_append(k.view(torch.int16).numpy(), v.view(torch.int16).numpy(), np.zeros((3, 16, 2, 128), np.int16),
                                np.zeros((3, 16, 2, 128), np.int16), slots[:entries].tolist(), rows[:entries].tolist())
        assert np.array_equal(kc.view(torch.int16).cpu().numpy(), wk) and status.item() == word
        assert np.array_equal(vc.view(torch.int16).cpu().numpy(), wv)


def test_append_views(cuda):
    """Rows off 16-byte alignment, rows that repeat one head, a cache inside a larger one; nothing beside a slot changes."""
    from dforktree_amd import ops
    announce("append views")
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(20, 2 * 128 * 2 + 3, generator=g).to(torch.bfloat16)
    slots = torch.randperm(48, generator=g)[:20]
    for at in (0, 1, 3):
        x = wide.to(cuda)
        k, v = x[:, at:at + 256].unflatten(1, (2, 128)), x[:, at + 256:at + 512].unflatten(1, (2, 128))
        shared = x[:, None, at:at + 128].expand(20, 2, 128)
        for kk, vv in ((k, v), (shared, v)):
            big = torch.full((3, 17, 3, 136), 5.0, device=cuda, dtype=torch.bfloat16)
            both = [big.clone()[:, 1:, 1:, 8:], big.clone()[:, 1:, 1:, 8:]]
            ops.kv_append(kk, vv, *both, slots.to(cuda))
            torch.cuda.synchronize()
            wk, wv, _ = P.kv_append(kk.float().cpu().numpy(), vv.float().cpu().numpy(), np.full((3, 16, 2, 128), 5.0),
                                    np.full((3, 16, 2, 128), 5.0), slots.tolist())
            for c, w in zip(both, (wk, wv)):
                assert np.array_equal(c.float().cpu().numpy(), w)
                whole = c._base if c._base is not None else c
                assert (whole[:, 0] == 5).all() and (whole[:, :, 0] == 5).all() and (whole[..., :8] == 5).all()


def test_far_slots(cuda):
    """A cache of over 2^32 elements."""
    from dforktree_amd import ops
    announce("far slots")
    pages = (1 << 32) // (16 * 2 * 128) + 3
    cache = torch.empty(pages, 16, 2, 128, dtype=torch.bfloat16, device=cuda)
    k = torch.randn(5, 2, 128, device=cuda).to(torch.bfloat16)
    slots = torch.tensor([pages * 16 - 1, pages * 16 - 17, 0, 5, pages * 8], device=cuda)
    ops.kv_append(k, k, cache, cache, slots)
    torch.cuda.synchronize()
    assert torch.equal(cache.view(-1, 2, 128)[slots], k)


def test_refusals(cuda):
    from dforktree_amd import ops
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    good = dict(prefix_len=i32(2), new_len=i32(2), block_table=i32(2, 3), held=i32(2), free_pages=i32(5),
                free_pos=torch.zeros(2, dtype=torch.int64, device=cuda), page_size=4, rows=3)
    ops.page_plan(**good)
    for bad, error in ((dict(new_len=i32(3)), ValueError), (dict(held=i32(1)), ValueError),
                       (dict(prefix_len=torch.zeros(2, device=cuda)), TypeError), (dict(held=i32(2).long()), TypeError),
                       (dict(block_table=i32(2, 3).long()), TypeError), (dict(block_table=i32(3, 2).t()), ValueError),
                       (dict(block_table=i32(6)), ValueError), (dict(block_table=i32(1, 3).expand(2, 3)), ValueError),
                       (dict(free_pages=i32(10)[::2]), ValueError), (dict(free_pages=i32(0)), ValueError),
                       (dict(free_pos=i32(2)), ValueError), (dict(page_size=0), ValueError), (dict(rows=-1), ValueError),
                       (dict(depth=i32(2)), ValueError), (dict(index_dtype=torch.float32), TypeError),
                       (dict(held=torch.zeros(2, dtype=torch.int32)), ValueError)):
        with pytest.raises(error):
            ops.page_plan(**(good | bad))
    x, c = torch.zeros(4, 2, 64, device=cuda), torch.zeros(3, 4, 2, 64, device=cuda)
    s = i32(4)
    for args, kw, error in (((x, x[:3], c, c, s), {}, ValueError), ((x, x.half(), c, c, s), {}, TypeError),
                            ((x, x, c, c[:2], s), {}, ValueError), ((x, x, c, c.half(), s), {}, TypeError),
                            ((x[:, :1], x[:, :1], c, c, s), {}, ValueError), ((x, x, c, c, i32(5)), {}, ValueError),
                            ((x, x, c, c, s.float()), {}, TypeError), ((x, x, c, c, s), dict(rows=i32(3)), ValueError),
                            ((x, x, c, c, s), dict(rows=s.float()), TypeError), ((x, x, c[0], c[0], s), {}, ValueError),
                            ((x.long(), x.long(), c, c, s), {}, TypeError),
                            ((x, x, c, c, s), dict(status=torch.zeros(1, device=cuda)), ValueError)):
        with pytest.raises(error):
            ops.kv_append(*args, **kw)
