"""Paged and prompt attention against a 64-bit softmax.

The bounds are counted, not fitted: with u the half step of the inputs' type
(the weights p are rounded to it before they multiply v), uo the output's, and
eps = (d + 8) 2^-24 |scale| max_j sum |q k_j| the error of a 32-bit score,

    |o - exact|   <= (u + 2 eps + (L + 64) 2^-24) sum_j p_j |v_j| + uo |o|
                     (+ L 2^-25 max |v| in fp16, whose weights below 2^-14 lose their relative precision)
    |lse - exact| <= eps + (L + 64) 2^-24 + 2^-22 |lse|
"""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def dense(q, k, v, sees, scale):
    """oracle.attend over whole matrices, for values without NaN or infinity (float64 tensors on the CPU)."""
    n, hq, d = q.shape
    o, lse = torch.zeros(n, hq, d, dtype=torch.float64), torch.full((n, hq), -np.inf, dtype=torch.float64)
    weight, reach = torch.zeros_like(o), torch.zeros(n, hq, dtype=torch.float64)
    sees = torch.as_tensor(sees)
    some = sees.any(1)
    if not some.any():
        return o, lse, weight, reach
    for h in range(hq):
        g = h * k.shape[1] // hq
        s = torch.where(sees, scale * (q[:, h] @ k[:, g].T), -np.inf)
        p = torch.where(some[:, None], torch.softmax(s, 1), 0)
        o[:, h], weight[:, h] = p @ v[:, g], p @ v[:, g].abs()
        lse[:, h] = torch.logsumexp(s, 1)
        reach[:, h] = torch.where(sees, abs(scale) * (q[:, h].abs() @ k[:, g].abs().T), 0).amax(1)
    return o, lse, weight, reach


def check(o, lse, exact, keys, dtype, vmax, what):
    eo, elset, weight, reach = (torch.as_tensor(x) for x in exact)
    d = eo.shape[-1]
    u, uo = torch.finfo(dtype).eps / 2, torch.finfo(o.dtype).eps / 2
    eps = (d + 8) * 2.0 ** -24 * reach
    rel = u + 2 * eps + (keys + 64) * 2.0 ** -24
    tol = rel[..., None] * weight + uo * eo.abs() + 1e-30
    if dtype == F16:
        tol += torch.where(torch.isfinite(elset), keys * 2.0 ** -25 * vmax, 0.0)[..., None]
    off = (o.double().cpu() - eo).abs()
    assert torch.isfinite(o).all(), f"{what}: {(~torch.isfinite(o)).sum()} outputs are not finite"
    assert (off <= tol).all(), f"{what}: off by {(off / tol).max():.2f} of the bound at {np.unravel_index(int((off / tol).argmax()), off.shape)}"
    if lse is not None:
        lse = lse.double().cpu()
        assert torch.equal(torch.isinf(lse), torch.isinf(elset)) and not torch.isnan(lse).any(), f"{what}: lse"
        ok = torch.isfinite(elset)
        off, tol = (lse - elset)[ok].abs(), (eps + (keys + 64) * 2.0 ** -24 + 2.0 ** -22 * elset.abs())[ok]
        assert (off <= tol).all(), f"{what}: lse off by {(off / tol).max():.2f} of the bound"


class Paged:
    """A batch over a cache that holds NaN wherever no token of it lives."""

    def __init__(self, cuda, seed, prefix, new, *, hq, hkv, d, ps, dtype=BF16, heads_first=False, qscale=1.0, spare=2,
                 poison=True, keys=None):
        g = torch.Generator().manual_seed(seed)
        self.prefix, self.new = prefix, new
        self.total = [p + n for p, n in zip(prefix, new)] if keys is None else keys
        held = [-(-max(t, 0) // ps) for t in self.total]
        pages = sum(held) + 3
        order = torch.randperm(pages, generator=g)
        shape = (pages, hkv, ps, d) if heads_first else (pages, ps, hkv, d)
        caches = [torch.full(shape, float("nan") if poison else 0.0, dtype=dtype) for _ in range(2)]
        self.k, self.v = (c.transpose(1, 2) if heads_first else c for c in caches)
        table = torch.randint(-5, pages + 5, (len(new), max(held, default=0) + spare), generator=g).int()  # junk past held
        at = 0
        for b, (h, t) in enumerate(zip(held, self.total)):
            table[b, :h] = order[at:at + h]
            at += h
            for c in (self.k, self.v):
                for j in range(h):
                    m = min(ps, t - j * ps)
                    c[table[b, j], :m] = torch.randn(m, hkv, d, generator=g).to(dtype)
        self.table = table
        self.rows = sum(new)
        self.q = (torch.randn(self.rows, hq, d, generator=g) * qscale).to(dtype)
        self.cu = torch.tensor([0, *np.cumsum(new)], dtype=torch.int32)
        self.ps, self.dtype, self.cuda = ps, dtype, cuda

    def gpu(self, t, dtype=None):
        return t.to(self.cuda) if dtype is None else t.to(self.cuda, dtype)

    def caches(self):
        if self.k.is_contiguous():
            return self.gpu(self.k), self.gpu(self.v)
        return tuple(self.gpu(c.transpose(1, 2).contiguous()).transpose(1, 2) for c in (self.k, self.v))

    def run(self, *, causal=True, bits=None, lse=True, scale=None, **kw):
        from dforktree_amd import ops
        k, v = self.caches()
        lse = torch.full(self.q.shape[:2], 7.0, device=self.cuda) if lse else None
        o = ops.paged_attention(self.gpu(self.q), k, v, self.gpu(self.table),
                                torch.tensor(self.total, dtype=torch.int32, device=self.cuda), cu_seqlens=self.gpu(self.cu),
                                n_new=max(self.new, default=0), causal=causal,
                                anc_bits=None if bits is None else self.gpu(bits), lse=lse, scale=scale, **kw)
        torch.cuda.synchronize()
        return o, lse

    def check(self, o, lse, *, causal=True, bits=None, scale=None, what="", slow=False):
        d = self.q.shape[2]
        scale = d ** -0.5 if scale is None else scale
        for b, (n, t) in enumerate(zip(self.new, self.total)):
            r0 = int(self.cu[b])
            k, there = P.paged_keys(self.k.float().numpy(), self.table[b].numpy(), t)
            v, _ = P.paged_keys(self.v.float().numpy(), self.table[b].numpy(), t)
            if bits is not None:
                sees = P.sees_tree(bits[r0:r0 + n].numpy(), t)
            elif causal:
                sees = P.sees_causal(n, t)
            else:
                sees = np.ones((n, t), bool)
            sees = sees & there
            q = self.q[r0:r0 + n].double()
            if slow:
                exact = P.attend(q.numpy(), k, v, sees, scale)
            else:
                exact = dense(q, torch.as_tensor(k).double(), torch.as_tensor(v).double(), sees, scale)
            vmax = float(np.abs(v[sees.any(0)]).max()) if sees.any() else 0.0
            check(o[r0:r0 + n], None if lse is None else lse[r0:r0 + n], exact, t, self.dtype, vmax, f"{what} request {b}")


def ancestry(sizes, seed):
    rng = np.random.default_rng(seed)
    words = []
    for n in sizes:
        bits = []
        for i in range(n):
            bits.append((bits[rng.integers(max(0, i - 5), i)] if i else 0) | 1 << i)
        words += bits
    return torch.from_numpy(np.array(words, np.uint64).view(np.int64))


HEADS = [(4, 4), (8, 2), (8, 1), (14, 2), (32, 8), (40, 1)]
EDGES = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_single_tokens(cuda, d, heads, dtype):
    """One new token each over prefixes at the tiles' edges, pages that end inside a tile."""
    announce(f"single tokens d={d} heads={heads} {dtype}")
    t = Paged(cuda, d + heads[0], [0, *EDGES, 700], [1] * (len(EDGES) + 2), hq=heads[0], hkv=heads[1], d=d, ps=24, dtype=dtype)
    t.check(*t.run(), what=f"d={d} {heads}")


@pytest.mark.parametrize("ps", [1, 3, 16, 64, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_page_sizes_and_layouts(cuda, ps, heads_first):
    announce(f"page size {ps}, heads first {heads_first}")
    t = Paged(cuda, ps, [0, 5, 63, 64, 300, 511], [1, 2, 1, 33, 70, 1], hq=8, hkv=2, d=128, ps=ps, heads_first=heads_first)
    t.check(*t.run(), what=f"ps={ps}")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (14, 2), (32, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chunks(cuda, d, heads, dtype):
    """Chunks of every size class, ragged, with empty requests between them."""
    announce(f"chunks d={d} heads={heads} {dtype}")
    t = Paged(cuda, 3, [0, 7, 100, 0, 64, 333, 31], [129, 0, 65, 1, 64, 17, 200], hq=heads[0], hkv=heads[1], d=d, ps=16,
              dtype=dtype)
    t.check(*t.run(), what=f"d={d} {heads}")
    t.check(*t.run(causal=False), causal=False, what=f"all d={d} {heads}")


@pytest.mark.parametrize("new", [2, 3, 5, 8, 9, 16, 24, 31, 40, 64])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1)])
def test_few_rows(cuda, new, heads):
    """Every count of packed query rows around the tile heights."""
    announce(f"few rows {new} heads={heads}")
    t = Paged(cuda, new, [0, 77, 200], [new, max(1, new - 1), new], hq=heads[0], hkv=heads[1], d=128, ps=16)
    t.check(*t.run(), what=f"new={new} {heads}")


@pytest.mark.parametrize("d,heads", [(64, (4, 4)), (128, (32, 8)), (128, (8, 1)), (256, (16, 2)), (256, (7, 1))])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_trees(cuda, d, heads, dtype):
    announce(f"trees d={d} heads={heads} {dtype}")
    sizes = [1, 8, 31, 32, 33, 63, 64, 0, 17]
    bits = ancestry(sizes, d)
    t = Paged(cuda, 5, [0, 1, 31, 100, 97, 63, 640, 9, 255], sizes, hq=heads[0], hkv=heads[1], d=d, ps=16, dtype=dtype)
    t.check(*t.run(bits=bits), bits=bits, what=f"trees d={d} {heads}")


def test_tree_rows_without_keys(cuda):
    """Words without bits, over an empty and a short prefix; bits past the tree are no tokens."""
    announce("tree rows without keys")
    sizes = [5, 40, 3]
    bits = ancestry(sizes, 0)
    bits[1] = bits[20] = bits[47] = 0
    bits[2] = -1  # every bit: the request has 5 tokens
    t = Paged(cuda, 1, [0, 0, 70], sizes, hq=8, hkv=2, d=128, ps=16)
    o, lse = t.run(bits=bits)
    assert (o[1] == 0).all() and torch.isinf(lse[1]).all() and (o[20] == 0).all()
    t.check(o, lse, bits=bits, what="empty words")


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_in_front_of_the_keys(cuda, d):
    """Fewer keys than rows (and none): the first rows see nothing."""
    announce(f"more rows than keys d={d}")
    t = Paged(cuda, 2, [0, 0, 0, 0], [70, 40, 3, 1], hq=8, hkv=2, d=d, ps=16, keys=[33, 0, 1, 0])
    o, lse = t.run()
    assert (o[:37] == 0).all() and (lse[:37] == -np.inf).all() and (o[70:110] == 0).all()
    t.check(o, lse, what="fewer keys than rows")


def test_long_and_ragged(cuda):
    """One long request beside short ones: its keys are split, theirs are not."""
    announce("long and ragged")
    t = Paged(cuda, 4, [9001, 3, 0, 130, 4100], [1] * 5, hq=8, hkv=2, d=128, ps=16)
    t.check(*t.run(), what="ragged")
    t = Paged(cuda, 5, [20011], [1], hq=16, hkv=2, d=256, ps=64, dtype=F16)
    t.check(*t.run(), what="long")
    t = Paged(cuda, 6, [5003, 40], [33, 64], hq=16, hkv=2, d=128, ps=1)
    bits = ancestry([33, 64], 3)
    t.check(*t.run(bits=bits), bits=bits, what="long trees")


def test_large_scores(cuda):
    """Scores of some hundreds: one key takes all; and a scale of zero: all share."""
    announce("large scores")
    t = Paged(cuda, 7, [500, 63], [9, 1], hq=8, hkv=2, d=128, ps=16, qscale=30.0)
    t.check(*t.run(), what="large")
    t = Paged(cuda, 7, [500, 63], [9, 1], hq=8, hkv=2, d=128, ps=16)
    t.check(*t.run(scale=0.0), scale=0.0, what="scale 0")
    t.check(*t.run(scale=-0.2), scale=-0.2, what="negative scale")


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_unseen_tokens_may_hold_anything(cuda, junk):
    """Values of new tokens that only later rows see do not reach earlier rows."""
    announce(f"unseen tokens {junk}")
    for d, heads, new in ((128, (4, 1), 40), (64, (4, 4), 130), (256, (8, 1), 9)):
        t = Paged(cuda, 8, [50], [new], hq=heads[0], hkv=heads[1], d=d, ps=16)
        tok = 50 + new - 3  # seen by the last three rows only
        page, at = int(t.table[0, tok // 16]), tok % 16
        t.v[page, at, 0, 5] = junk
        o, lse = t.run()
        kept, exact_lse = o[:new - 3], lse[:new - 3]
        sees = P.sees_causal(new, 50 + new)[:new - 3]
        k, _ = P.paged_keys(t.k.float().numpy(), t.table[0].numpy(), 50 + new)
        v, _ = P.paged_keys(t.v.float().numpy(), t.table[0].numpy(), 50 + new)
        exact = P.attend(t.q[:new - 3].double().numpy(), k, v, sees, d ** -0.5)
        check(kept, exact_lse, exact, 50 + new, BF16, 10.0, f"{junk} d={d}")
        bad = o[new - 3:].float()
        per = heads[0] // heads[1]
        assert not torch.isfinite(bad[:, :per, 5]).any()
        assert torch.isfinite(bad[:, :per, 6]).all() and torch.isfinite(bad[:, :per, 4]).all()
        t.k[page, at, 0, 5] = junk
        t.v[page, at, 0, 5] = 1.0
        o, lse = t.run()
        check(o[:new - 3], lse[:new - 3], exact, 50 + new, BF16, 10.0, f"key {junk} d={d}")


def test_pages_outside_the_cache(cuda):
    """Bad page ids inside a request's range hold no keys; too few columns cut it."""
    from dforktree_amd import _lib
    announce("bad pages")
    t = Paged(cuda, 9, [200, 333, 90], [4, 33, 1], hq=8, hkv=2, d=128, ps=16, spare=0)
    t.table[0, 3], t.table[1, 0], t.table[1, 7] = -1, 1 << 30, t.k.shape[0]
    t.table[2, :6] = -7
    status = torch.full((3,), 99, dtype=torch.int32, device=cuda)
    o, lse = t.run(status=status)
    assert status.tolist() == [0, 0, 0]
    t.check(o, lse, what="bad pages")
    # a length past the table: the rows of request 0 see what the table holds, the other requests stay as they were
    t.k.nan_to_num_(0.0)
    t.v.nan_to_num_(0.0)
    old = t.total[0]
    t.total[0] = 2000
    again, again_lse = t.run(status=status)
    assert status.tolist() == [_lib.DFT_STATUS_TABLE, 0, 0]
    assert torch.equal(again[4:], o[4:]) and torch.equal(again_lse[4:], lse[4:])
    t.check(again, again_lse, what="past the table")
    assert old < 2000


def test_spans_that_do_not_fit(cuda):
    """Requests longer than n_new, negative, or past the rows are cut and marked."""
    from dforktree_amd import _lib, ops
    announce("spans")
    t = Paged(cuda, 10, [20, 30, 40], [5, 6, 7], hq=8, hkv=2, d=64, ps=16)
    k, v = t.caches()
    status = torch.full((3,), 99, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 5, 11, 40], dtype=torch.int32, device=cuda)
    o = torch.full(t.q.shape, 7.0, dtype=BF16, device=cuda)
    ops.paged_attention(t.gpu(t.q), k, v, t.gpu(t.table), torch.tensor(t.total, device=cuda), cu_seqlens=cu, n_new=5, o=o,
                        status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, _lib.DFT_STATUS_SPAN, _lib.DFT_STATUS_SPAN]
    assert (o[10] == 7).all() and (o[16:] == 7).all() and (o[:10] != 7).all(-1).all() and (o[11:16] != 7).any()
    cu = torch.tensor([0, 5, 3, 10], dtype=torch.int32, device=cuda)
    ops.paged_attention(t.gpu(t.q), k, v, t.gpu(t.table), torch.tensor(t.total, device=cuda), cu_seqlens=cu, n_new=7, o=o,
                        status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, _lib.DFT_STATUS_SPAN, 0]


def test_views_types_and_uniform_batches(cuda):
    """Sliced queries, outputs inside a larger buffer, fp32 outputs, an int64 seq_len, rows without cu_seqlens."""
    from dforktree_amd import ops
    announce("views")
    t = Paged(cuda, 11, [33, 100, 64], [4, 4, 4], hq=8, hkv=2, d=128, ps=16)
    k, v = t.caches()
    for pad in (8, 3):  # 3: rows that are not 16-byte aligned
        wide = torch.randn(12, 8 * 128 + pad + 64, device=cuda).to(BF16)
        q = wide[:, pad:pad + 1024].unflatten(1, (8, 128))
        t.q = q.cpu()
        for od in (BF16, F16, F32):
            big = torch.full((13, 9, 140), 7.0, device=cuda, dtype=od)
            o = big[1:, 1:, 5:133]
            table = torch.full((3, 40), -1, dtype=torch.int32, device=cuda)[:, ::2]
            table[:, :t.table.shape[1]] = t.gpu(t.table)[:, :20]
            r = ops.paged_attention(q, k, v, table, torch.tensor(t.total, device=cuda), n_new=4, o=o)
            torch.cuda.synchronize()
            assert r is o and (big[0] == 7).all() and (big[:, 0] == 7).all() and (big[..., :5] == 7).all()
            assert (big[..., 133:] == 7).all()
            t.check(o, None, what=f"views pad={pad} {od}")


def test_repeatable_and_on_other_streams(cuda):
    """The same bits every time, on the current stream whatever it is."""
    announce("streams")
    from dforktree_amd import ops
    t = Paged(cuda, 12, [3000, 5, 900], [3, 40, 1], hq=8, hkv=2, d=128, ps=16)
    first, lse = t.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k, v = t.caches()
        args = (t.gpu(t.q), k, v, t.gpu(t.table), torch.tensor(t.total, device=cuda))
        again = [ops.paged_attention(*args, cu_seqlens=t.gpu(t.cu), n_new=40) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(first, x) for x in again)


def test_in_a_graph(cuda):
    """Captured once; replays follow the lengths and pages that the buffers hold."""
    announce("graph")
    from dforktree_amd import ops
    t = Paged(cuda, 13, [2500, 77, 130], [1, 1, 1], hq=8, hkv=2, d=128, ps=16)
    k, v = t.caches()
    q, table, cu = t.gpu(t.q), t.gpu(t.table), t.gpu(t.cu)
    total = torch.tensor(t.total, dtype=torch.int32, device=cuda)
    o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=cuda)
    call = lambda: ops.paged_attention(q, k, v, table, total, cu_seqlens=cu, n_new=1, o=o, lse=lse)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for lengths in ([2501, 78, 131], [1000, 1, 131], [0, 78, 5], [2501, 78, 131]):
        total.copy_(torch.tensor(lengths))
        t.total = lengths
        o.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.check(o, lse, what=f"replay {lengths}")


def test_far_pages(cuda):
    """Offsets past 32 bits: the pages lie at the end of a buffer of over 2^32 elements."""
    announce("far pages")
    from dforktree_amd import ops
    t = Paged(cuda, 14, [100, 64], [1, 20], hq=8, hkv=2, d=128, ps=16, poison=False)
    pages = t.k.shape[0]
    page = 16 * 2 * 128
    far = (1 << 32) // page + 5
    both = torch.empty(2, far + pages, 16, 2, 128, dtype=BF16, device=cuda)
    both[0, far:], both[1, far:] = t.gpu(t.k), t.gpu(t.v)
    table = torch.where(t.table >= 0, t.table + far, -1)
    o = ops.paged_attention(t.gpu(t.q), both[0], both[1], t.gpu(table), torch.tensor(t.total, device=cuda),
                            cu_seqlens=t.gpu(t.cu), n_new=20)
    t.check(o, None, what="far")
    # and as strides: two caches interleaved page by page
    del both
    torch.cuda.empty_cache()


# ---- prompts ----------------------------------------------------------------
def prompt(cuda, sizes, hq, hkv, d, dtype, *, causal=True, seed=0, scale=None, junk=None, **kw):
    from dforktree_amd import ops
    g = torch.Generator().manual_seed(seed)
    rows = sum(sizes)
    qkv = torch.randn(rows, hq + 2 * hkv, d, generator=g).to(dtype)
    if junk:
        junk(qkv)
    x = qkv.to(cuda)
    cu = torch.tensor([0, *np.cumsum(sizes)], dtype=torch.int32, device=cuda)
    lse = torch.full((rows, hq), 7.0, device=cuda)
    o = ops.prompt_attention(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], cu, max_len=max(sizes), causal=causal, lse=lse,
                             scale=scale, **kw)
    torch.cuda.synchronize()
    return qkv, o, lse


def check_prompt(qkv, o, lse, sizes, hq, hkv, d, dtype, *, causal=True, scale=None, what=""):
    at = 0
    for n in sizes:
        x = qkv[at:at + n].double()
        sees = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
        exact = dense(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], sees, d ** -0.5 if scale is None else scale)
        check(o[at:at + n], lse[at:at + n], exact, n, dtype, float(x[:, hq + hkv:].abs().max()) if n else 0.0,
              f"{what} prompt of {n}")
        at += n


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(cuda, d, heads, dtype, causal):
    """Packed lengths at the tiles' edges, empty ones among them."""
    sizes = [1, 0, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 200, 257, 2]
    announce(f"prompts d={d} heads={heads} {dtype} causal={causal}")
    r = prompt(cuda, sizes, *heads, d, dtype, causal=causal, seed=d)
    check_prompt(*r, sizes, *heads, d, dtype, causal=causal, what=f"d={d} {heads}")


@pytest.mark.parametrize("d,heads,n", [(128, (8, 2), 1500), (64, (2, 2), 2049), (256, (4, 1), 1023)])
def test_long_prompts(cuda, d, heads, n):
    announce(f"long prompts d={d} {heads} {n}")
    r = prompt(cuda, [n, 5], *heads, d, BF16, seed=1)
    check_prompt(*r, [n, 5], *heads, d, BF16, what=f"long d={d}")


def test_prompt_scores_that_grow(cuda):
    """Later keys score ever higher, so the running maximum moves in every tile; and far below it."""
    announce("growing scores")

    def grow(qkv):
        ramp = torch.linspace(-12, 12, qkv.shape[0])[:, None]
        qkv[:, 4] = (ramp * torch.ones(64)).to(BF16)   # k of the one kv head
        qkv[:, :2] = qkv[:, :2].abs()
        qkv[:, 2:4] = -qkv[:, 2:4].abs()

    r = prompt(cuda, [400], 4, 1, 64, BF16, junk=grow)
    check_prompt(*r, [400], 4, 1, 64, BF16, what="growing")


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_prompt_tokens_ahead_may_hold_anything(cuda, junk):
    announce(f"tokens ahead {junk}")
    for d, n, at in ((128, 150, 141), (64, 70, 40), (256, 90, 89)):
        clean = prompt(cuda, [n, 20], 4, 2, d, BF16, seed=2)

        def spoil(qkv):
            qkv[at, 6:, 3] = junk    # v
            qkv[at, 4:6, 7] = junk   # k

        _, o, lse = prompt(cuda, [n, 20], 4, 2, d, BF16, seed=2, junk=spoil)
        assert torch.equal(o[:at], clean[1][:at]) and torch.equal(lse[:at], clean[2][:at])
        assert torch.equal(o[n:], clean[1][n:])
        assert not torch.isfinite(o[at:n]).all()


def test_prompts_without_cu_seqlens_and_cut(cuda):
    from dforktree_amd import _lib, ops
    announce("uniform prompts")
    x = torch.randn(60, 8, 64, device=cuda).to(BF16)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    cu = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=cuda)
    want = ops.prompt_attention(q, k, v, cu, max_len=20)
    assert torch.equal(ops.prompt_attention(q, k, v, max_len=20), want)
    assert torch.equal(ops.prompt_attention(q, k, v, batch=3), want)
    one = ops.prompt_attention(q[:20], k[:20], v[:20])
    assert torch.equal(one, want[:20])
    status = torch.full((3,), 9, dtype=torch.int32, device=cuda)
    o = torch.full((60, 4, 64), 7.0, device=cuda, dtype=BF16)
    ops.prompt_attention(q, k, v, torch.tensor([0, 20, 45, 77], dtype=torch.int32, device=cuda), max_len=20, o=o, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, _lib.DFT_STATUS_SPAN, _lib.DFT_STATUS_SPAN]
    assert torch.equal(o[:20], want[:20]) and (o[40:45] == 7).all() and (o[45:] != 7).any()
    assert ops.prompt_attention(q[:0], k[:0], v[:0], cu[:1], max_len=0).shape == (0, 4, 64)


def test_prompts_in_a_graph_and_repeatable(cuda):
    from dforktree_amd import ops
    announce("prompt graph")
    x = torch.randn(300, 8, 128, device=cuda).to(BF16)
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=cuda)
    call = lambda: ops.prompt_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu, max_len=300)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = call()
    for step in range(3):
        cu.copy_(torch.tensor([0, 100 - step, 300]))
        want = call()
        torch.cuda.synchronize()
        o.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


def test_refusals(cuda):
    from dforktree_amd import ops
    from dforktree_amd._lib import DftError
    q, k = torch.zeros(4, 4, 128, device=cuda, dtype=BF16), torch.zeros(4, 2, 128, device=cuda, dtype=BF16)
    cache = torch.zeros(3, 16, 2, 128, device=cuda, dtype=BF16)
    table, total = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    paged = lambda q=q, kc=cache, vc=cache, table=table, total=total, **kw: ops.paged_attention(  # noqa: E731
        q, kc, vc, table, total, **kw)
    for f, error in (
            (lambda: paged(q=q.float()), TypeError), (lambda: paged(q=q.half()), TypeError),
            (lambda: paged(vc=cache.half()), TypeError), (lambda: paged(kc=cache[:2]), ValueError),
            (lambda: paged(q=q[:, :3]), ValueError), (lambda: paged(q=q[..., :64]), ValueError),
            (lambda: paged(q=q[0]), ValueError), (lambda: paged(table=table.long()), TypeError),
            (lambda: paged(table=table[0]), ValueError), (lambda: paged(total=total.float()), TypeError),
            (lambda: paged(cu_seqlens=cu), ValueError), (lambda: paged(cu_seqlens=cu.long(), n_new=4), TypeError),
            (lambda: paged(cu_seqlens=cu[:1], n_new=4), ValueError), (lambda: paged(n_new=5), ValueError),
            (lambda: paged(anc_bits=torch.zeros(3, dtype=torch.int64, device=cuda)), ValueError),
            (lambda: paged(anc_bits=torch.zeros(4, dtype=torch.int32, device=cuda)), TypeError),
            (lambda: paged(o=q[:2]), ValueError), (lambda: paged(lse=q[..., 0]), TypeError),
            (lambda: paged(lse=torch.zeros(4, 5, device=cuda)), ValueError),
            (lambda: paged(status=torch.zeros(0, dtype=torch.int32, device=cuda)), ValueError),
            (lambda: paged(kc=cache.transpose(2, 3), vc=cache.transpose(2, 3)), ValueError),
            (lambda: paged(q=q[..., :72], kc=cache[..., :72], vc=cache[..., :72]), DftError),
            (lambda: paged(kc=cache[..., 4:68], vc=cache[..., 4:68], q=q[..., :64]), DftError),
            (lambda: ops.prompt_attention(q, k, k[:3]), ValueError),
            (lambda: ops.prompt_attention(q, k.half(), k), TypeError),
            (lambda: ops.prompt_attention(q[:, :3], k, k), ValueError),
            (lambda: ops.prompt_attention(q, k, k, cu), ValueError),
            (lambda: ops.prompt_attention(q, k, k, batch=2, max_len=3), ValueError),
            (lambda: ops.prompt_attention(q.float(), k.float(), k.float()), TypeError),
            (lambda: ops.prompt_attention(q[..., :32], k[..., :32], k[..., :32]), DftError)):
        with pytest.raises(error):
            f()
    big = torch.zeros(65, 4, 128, device=cuda, dtype=BF16)
    with pytest.raises(ValueError, match="64 nodes"):
        paged(q=big, anc_bits=torch.zeros(65, dtype=torch.int64, device=cuda))
