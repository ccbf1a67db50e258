"""A GDN layer's requests from their prompts over draft trees to single tokens, the operators together as a server runs
them, beside one full-attention layer's cache."""
import numpy as np
import pytest
import torch

from conftest import announce, rel_l2
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_from_prompt_to_tokens(cuda):
    """Every request's GDN state and window against the 64-bit recurrence over the tokens that it was left with.

    The convolution's outputs are rounded to bf16 in between, in the oracle from its own 64 bits: where the two round a
    value apart (a share of 2^-15 or so of them: both are within 16 * 2^-24 of each other, a step is 2^-8) a row is a
    step off, 2^-8 of one of 128 values.  So the state is held to 2^-11 in the 2-norm here."""
    from dforktree_amd import ops
    from dforktree_amd.paged import PagedKV
    announce("from prompt to tokens")
    rng, g = np.random.default_rng(0), torch.Generator().manual_seed(0)
    B, hk, hv, V, ahead = 3, 1, 2, 50, 12
    C = (2 * hk + hv) * 128
    embed = torch.randn(V, C, generator=g).to(BF16).to(cuda)  # a token's projection in front of the convolution
    gates = torch.randn(V, 2 * hv, generator=g).to(BF16).to(cuda)
    heads = torch.randn(hv * 128, V, generator=g).to(cuda) * 0.15
    kv_rows = torch.randn(V, 2, 2, 64, generator=g).to(BF16).to(cuda)
    w, bias = (torch.randn(C, 4, generator=g) * 0.5).to(BF16).to(cuda), torch.randn(C, generator=g).to(BF16).to(cuda)
    A_log, dt = torch.zeros(hv, device=cuda), torch.full((hv,), -2.0, device=cuda)
    window, pool = torch.randn(B, C, 3, device=cuda).to(BF16), torch.randn(B, hv, 128, 128, device=cuda)
    S = pool.transpose(-1, -2)
    kv = PagedKV(1, B, 20, 3 * 20, 16, 2, 64, device=cuda)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    fresh = torch.zeros(B, dtype=torch.bool, device=cuda)
    history = [rng.integers(0, V, n).tolist() for n in (70, 5, 129)]

    def attend(plan, tokens):
        x = kv_rows[tokens]
        kv.append(0, x[:, 0], x[:, 1], plan)
        return x

    def gdn(tokens, cu, limit, **kw):
        y = ops.prompt_conv(embed[tokens], window, w, bias, cu, max_len=limit, batch=None if cu is not None else B, **kw)
        ab = gates[tokens]
        if cu is None:
            return ops.token_gdn(y, ab[:, :hv], ab[:, hv:], A_log, dt, S, hk=hk, hv=hv, **kw)
        return ops.prompt_gdn(y, ab[:, :hv], ab[:, hv:], A_log, dt, S, cu, hk=hk, hv=hv, max_len=limit, **kw)

    def settled():
        """The states after the tokens so far, by the oracle."""
        for b, tokens in enumerate(history):
            x = embed[tokens].double().cpu().numpy()
            y, left, _, _ = P.prompt_conv(x, np.zeros((1, C, 3)), w.double().cpu().numpy(), bias.double().cpu().numpy(), None,
                                          batch=1, limit=len(tokens))
            ab = gates[tokens].double().cpu().numpy()
            y = torch.from_numpy(y).to(BF16).double().numpy()
            _, want, _ = P.prompt_gdn(y, ab[:, :hv], ab[:, hv:], -np.ones(hv), np.full(hv, -2.0), np.zeros((1, hv, 128, 128)),
                                      None, hk=hk, hv=hv, batch=1, limit=len(tokens))
            assert rel_l2(S[b].cpu(), want[0]) <= 2.0 ** -11, (b, rel_l2(S[b].cpu(), want[0]))
            assert np.array_equal(window[b].double().cpu().numpy(), left[0])
            assert int(kv.prefix[b]) == len(tokens)
            slots = [int(kv.block_table[b, t // 16]) * 16 + t % 16 for t in range(len(tokens))]
            assert torch.equal(kv.keys[0].flatten(0, 1)[slots], kv_rows[tokens][:, 0])

    # the prompts, the longest in two pieces
    for pieces, new in (([h[:100] for h in history], fresh), ([h[100:] for h in history], ~fresh)):
        sizes = [len(p) for p in pieces]
        tokens = torch.tensor(sum(pieces, []), device=cuda)
        plan = kv.plan(ints(sizes), rows=sum(sizes), n_new=max(sizes))
        attend(plan, tokens)
        o = gdn(tokens, plan["cu_seqlens"], max(sizes), initial=new)
        kv.commit(ints(sizes))
    settled()

    # draft trees: the root is the last token that stands, drawn but not yet passed through the layers
    root = rng.integers(0, V, B).tolist()
    for step in range(3):
        sizes = [int(n) for n in rng.integers(2, ahead + 1, B)]
        parents = [[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, n)] for n in sizes]
        cu, T = ints([0, *np.cumsum(sizes)]), sum(sizes)
        parent = ints(sum(parents, []))
        tokens = torch.tensor(sum(([r] + rng.integers(0, V, n - 1).tolist() for r, n in zip(root, sizes)), []), device=cuda)
        ts = ops.tree_struct(parent, 4, cu_seqlens=cu, n_nodes=max(sizes), want=("anc_bits", "depth", "cidx"))
        plan = kv.plan(ints(sizes), rows=T, n_new=max(sizes), depth=ts["depth"], anc_bits=ts["anc_bits"], trim=True)
        x = attend(plan, tokens)
        # the layers' convolution and verify, a request at a time where the convolution takes trees of one size
        y = torch.empty(T, C, dtype=BF16, device=cuda)
        for b in range(B):
            r = slice(int(cu[b]), int(cu[b + 1]))
            y[r] = ops.tree_conv(embed[tokens[r]], window[b], w, bias, ts["cidx"][r].contiguous())[0]
        k, v, gain = (torch.zeros(1, hv, T, *d, device=cuda) for d in ((128,), (128,), ()))
        ab = gates[tokens]
        o = ops.tree_verify(y, ab[:, :hv], ab[:, hv:], A_log, dt, S, hk=hk, hv=hv, anc_bits=ts["anc_bits"], cu_seqlens=cu,
                            n_nodes=max(sizes), aux_k=k[0], aux_v=v[0], aux_g=gain[0])
        probs = torch.softmax(o.float().flatten(1) @ heads, 1)
        draft = torch.full_like(probs, 1 / V) if step % 2 else None
        got = ops.tree_accept(tokens, parent, probs, torch.rand(T, generator=g).to(cuda) * 0.1, torch.rand(B, generator=g).to(cuda),
                              draft_probs=draft, cu_seqlens=cu, n_nodes=max(sizes))
        # what stands goes into the states, the cache and the windows
        ops.tree_commit(pool.unsqueeze(0), k, v, gain, got["path"], n_nodes=max(sizes), cu_seqlens=cu)
        kv.accept(0, x[:, 0], x[:, 1], plan, got["rows"])
        kv.commit(got["path_len"])
        accepted = [tokens[r[r >= 0]].tolist() for r in got["rows"]]
        flat = torch.tensor(sum(accepted, []), device=cuda)
        ops.prompt_conv(embed[flat], window, w, bias, ints([0, *np.cumsum([len(t) for t in accepted])]), max_len=16)
        for h, t in zip(history, accepted):
            h += t
        root = got["token"].tolist()
        assert all(0 <= t < V for t in root)
        settled()
    assert any(len(t) > 1 for t in accepted) or int(got["path_len"].max()) >= 1

    # without drafts: a token each
    for _ in range(3):
        tokens = torch.tensor(root, device=cuda)
        plan = kv.plan(ints([1] * B), rows=B, n_new=1)
        attend(plan, tokens)
        o = gdn(tokens, None, 1)
        kv.commit(ints([1] * B))
        for h, t in zip(history, root):
            h.append(t)
        alone = torch.softmax(o.float().flatten(1) @ heads, 1)  # trees of a root alone: the next token's draw
        root = ops.tree_accept(tokens, torch.full((B,), -1, dtype=torch.int32, device=cuda), alone, torch.rand(B, device=cuda),
                               torch.rand(B, generator=g).to(cuda), n_nodes=1, batch=B)["token"].tolist()
    settled()
