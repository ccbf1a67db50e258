"""A serving loop over PagedKV: prompts, draft trees with accepted paths, single tokens, a finished request."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def tree(n, rng):
    return [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)]


@pytest.mark.parametrize("page_size,hq,hkv,d", [(1, 8, 2, 128), (16, 4, 4, 64), (24, 16, 2, 256)])
def test_serving_loop(cuda, page_size, hq, hkv, d):
    """Every attention of the loop against the oracle's over the tokens that were committed so far.

    The tolerance is that of the kernels' own tests for bf16: half a step (2^-8) of the weights and of the output,
    twice over the largest value, as the oracle rounds neither."""
    from dforktree_amd import ops
    from dforktree_amd.paged import PagedKV
    announce(f"serving loop page={page_size} hq={hq} hkv={hkv} d={d}")
    rng, g = np.random.default_rng(d), torch.Generator().manual_seed(d)
    B, layers = 3, 2
    columns = 200 // page_size + 1
    kv = PagedKV(layers, B, columns, B * columns, page_size, hkv, d, device=cuda)
    history = [[np.zeros((0, 2, hkv, d)) for _ in range(B)] for _ in range(layers)]

    def step(new, depth=None, bits=None, **kw):
        rows, ints = sum(new), lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        plan = kv.plan(ints(new), rows=rows, n_new=max(new), depth=depth, anc_bits=bits, **kw)
        assert not plan["status"].any()
        cu, fed = plan["cu_seqlens"].tolist(), []
        for layer in range(layers):
            qkv = torch.randn(rows, hq + 2 * hkv, d, generator=g).to(BF16)
            x = qkv.to(cuda)
            q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
            kv.append(layer, k, v, plan)
            o = kv.attend(layer, q, plan).double().cpu().numpy()
            host = qkv.double().numpy()
            for b in range(B):
                r = slice(cu[b], cu[b + 1])
                if not new[b]:
                    continue
                own = np.stack([host[r, hq:hq + hkv], host[r, hq + hkv:]], 1)
                keys = np.concatenate([history[layer][b], own])
                n, t = new[b], len(keys)
                sees = P.sees_causal(n, t) if bits is None else P.sees_tree(bits[r].cpu().numpy(), t)
                want = P.attend(host[r, :hq], keys[:, 0], keys[:, 1], sees, d ** -0.5)[0]
                assert np.abs(o[r] - want).max() <= 2 * 2.0 ** -8 * np.abs(keys[:, 1]).max()
            fed.append((k, v, host, cu))
        return plan, fed

    def keep(fed, b, rows, layer):
        host = fed[layer][2]
        history[layer][b] = np.concatenate([history[layer][b], np.stack([host[rows, hq:hq + hkv], host[rows, hq + hkv:]], 1)])

    prompts = [40, 1, 70]
    plan, fed = step(prompts)
    kv.commit(torch.tensor(prompts, dtype=torch.int32, device=cuda))
    for layer in range(layers):
        for b in range(B):
            keep(fed, b, np.arange(*fed[0][3][b:b + 2]), layer)
    for sizes in ([9, 16, 5], [20, 3, 12]):
        parents = [tree(n, rng) for n in sizes]
        cu = torch.tensor([0, *np.cumsum(sizes)], dtype=torch.int32, device=cuda)
        ts = ops.tree_struct(torch.tensor(sum(parents, []), device=cuda), 1, cu_seqlens=cu, n_nodes=max(sizes),
                             want=("anc_bits", "depth"))
        plan, fed = step(sizes, depth=ts["depth"], bits=ts["anc_bits"], trim=True)
        path = np.full((B, 8), -1)
        for b, p in enumerate(parents):  # from some node up to the root
            node, up = int(rng.integers(len(p))), []
            while node >= 0 and len(up) < 8:
                up.append(node)
                node = p[node]
            up = up[::-1] if node < 0 else [0]
            path[b, :len(up)] = int(cu[b]) + np.array(up)
        rows = torch.tensor(path, device=cuda)
        for layer in range(layers):
            kv.accept(layer, *fed[layer][:2], plan, rows)
            for b in range(B):
                keep(fed, b, path[b][path[b] >= 0], layer)
        kv.commit((rows >= 0).sum(1).int())
    plan, fed = step([1, 1, 1], trim=True)
    kv.commit(torch.ones(B, dtype=torch.int32, device=cuda))
    # the first request ends: its pages return, the others go on
    held = int(kv.held[0])
    kv.prefix[0] = 0
    before = kv.free_pos.tolist()
    for layer in range(layers):
        for b in range(B):
            keep(fed, b, np.arange(b, b + 1), layer)
        history[layer][0] = history[layer][0][:0]
    step([0, 2, 1], trim=True)
    assert int(kv.held[0]) == 0 and kv.free_pos[1] - before[1] >= held


def test_replayed_steps(cuda):
    """A decode step captured once: every replay takes the next token, and pages when it needs one."""
    from dforktree_amd.paged import PagedKV
    announce("replayed steps")
    B, hq, hkv, d, ps = 2, 4, 2, 64, 4
    kv = PagedKV(1, B, 8, 16, ps, hkv, d, device=cuda)
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(B, hq + 2 * hkv, d, dtype=BF16, device=cuda)
    one = torch.ones(B, dtype=torch.int32, device=cuda)

    def step():
        plan = kv.plan(one, rows=B, n_new=1)
        kv.append(0, x[:, hq:hq + hkv], x[:, hq + hkv:], plan)
        o = kv.attend(0, x[:, :hq], plan)
        kv.commit(one)
        return o

    seen = []
    for replay in range(12):
        host = torch.randn(B, hq + 2 * hkv, d, generator=g).to(BF16)
        seen.append(host.double().numpy())
        x.copy_(host)
        if replay == 0:
            o = step()  # eager
        elif replay == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o = step()
        if replay:
            torch.cuda.synchronize()
            graph.replay()
        torch.cuda.synchronize()
        assert kv.prefix.tolist() == [replay + 1] * B and kv.held.tolist() == [replay // ps + 1] * B
        past = np.stack(seen, 1)  # [B, tokens, heads, d]
        for b in range(B):
            sees = np.ones((1, replay + 1), bool)
            want = P.attend(past[b, -1:, :hq], past[b, :, hq:hq + hkv], past[b, :, hq + hkv:], sees, d ** -0.5)[0]
            off = np.abs(o[b:b + 1].double().cpu().numpy() - want).max()
            assert off <= 2 * 2.0 ** -8 * np.abs(past[b, :, hq + hkv:]).max()
