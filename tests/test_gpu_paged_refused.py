"""A serving loop over PagedKV whose pages run out and come back, eager and as replays of one captured step."""
import numpy as np
import pytest
import torch

from conftest import announce
from oracle import paged as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("page_size,hq,hkv,d", [(1, 8, 2, 128), (4, 4, 4, 64)])
def test_pages_run_out_and_return(cuda, captured, page_size, hq, hkv, d):
    """One token each a step.  The pool holds 8 pages for three requests: all of them stop growing when it is empty,
    and go on when the one that ends has returned its pages.  Every attention is compared with the oracle's over the
    tokens that the plan served; the bound is the serving loop's, half a step of bf16 (2^-8) of the weights and of the
    output, twice over the largest value."""
    from dforktree_amd.paged import PagedKV
    announce(f"pages run out: page={page_size} captured={captured}")
    B, pages, columns = 3, 8, 8
    kv = PagedKV(1, B, columns, pages, page_size, hkv, d, device=cuda)
    g = torch.Generator().manual_seed(page_size)
    x = torch.zeros(B, hq + 2 * hkv, d, dtype=BF16, device=cuda)
    new = torch.ones(B, dtype=torch.int32, device=cuda)
    mine = dict(prefix=np.zeros(B, int), table=np.full((B, columns), -1, np.int32), held=np.zeros(B, int),
                ring=np.arange(pages, dtype=np.int32), pos=np.array([0, pages]))
    history = [np.zeros((0, 2, hkv, d)) for _ in range(B)]

    def step():
        plan = kv.plan(new, rows=B, n_new=1, trim=True)
        kv.append(0, x[:, hq:hq + hkv], x[:, hq + hkv:], plan)
        o = kv.attend(0, x[:, :hq], plan)
        kv.commit(new)
        return o, plan["status"]

    refused = resumed = 0
    for at in range(12 * page_size):
        asked = [1, 1, 1]
        if at >= 6 * page_size:  # the second request has ended
            asked[1] = 0
        if at == 6 * page_size:
            kv.prefix[1], mine["prefix"][1], history[1] = 0, 0, history[1][:0]
        new.copy_(torch.tensor(asked))
        host = torch.randn(B, hq + 2 * hkv, d, generator=g).to(BF16)
        x.copy_(host)
        if not captured or at == 0:
            o, status = step()
        elif at == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o, status = step()
        if captured and at:
            torch.cuda.synchronize()
            graph.replay()
        torch.cuda.synchronize()
        r = P.page_plan(mine["prefix"], asked, mine["table"], mine["held"], mine["ring"], mine["pos"], page_size=page_size,
                        rows=B, trim=True)
        mine |= dict(table=r["block_table"], held=r["held"], ring=r["free_pages"], pos=r["free_pos"])
        assert status.tolist() == r["status"].tolist()
        host = host.double().numpy()
        for b in range(B):
            row = int(r["cu_seqlens"][b])
            if r["status"][b] & P.STATUS_PAGES:
                refused += 1
                assert (o[row] == 0).all()
            elif asked[b]:
                resumed += refused > 0
                mine["prefix"][b] += 1
                history[b] = np.concatenate([history[b], np.stack([host[row:row + 1, hq:hq + hkv], host[row:row + 1, hq + hkv:]], 1)])
                k, v = history[b][:, 0], history[b][:, 1]
                want = P.attend(host[row:row + 1, :hq], k, v, np.ones((1, len(k)), bool), d ** -0.5)[0]
                assert np.abs(o[row].double().cpu().numpy() - want[0]).max() <= 2 * 2.0 ** -8 * np.abs(v).max()
        assert kv.prefix.tolist() == mine["prefix"].tolist() == [len(h) for h in history]
        assert kv.held.tolist() == mine["held"].tolist() and kv.free_pos.tolist() == mine["pos"].tolist()
    assert refused and resumed
