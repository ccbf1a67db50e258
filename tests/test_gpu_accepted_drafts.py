"""Draft trees of which some nodes stand, step after step: the path that tree_accept finds, committed, leaves every
request's state and window where its tokens one after the other lead."""
import numpy as np
import pytest
import torch

from conftest import announce, rel_l2
from oracle import packed as P

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("drawn", [False, True])
def test_steps_with_accepted_drafts(cuda, drawn):
    """The convolution's outputs round to bf16 in between, in the oracle from its own 64 bits: a share of 2^-15 or so of
    them a step apart, 2^-8 of one of 128 values.  So states are held to 2^-11 in the 2-norm."""
    from dforktree_amd import ops
    announce(f"steps with accepted drafts, drawn={drawn}")
    rng, g = np.random.default_rng(5), torch.Generator().manual_seed(5)
    B, hk, hv, V = 3, 1, 2, 20
    C = (2 * hk + hv) * 128
    r = lambda *s: torch.randn(*s, generator=g).to(cuda)  # noqa: E731
    embed, gates, heads = r(V, C).to(BF16), r(V, 2 * hv).to(BF16), r(hv * 128, V) * 0.1
    w, bias = (r(C, 4) * 0.5).to(BF16), r(C).to(BF16)
    A_log, dt = torch.zeros(hv, device=cuda), torch.full((hv,), -2.0, device=cuda)
    window, pool = torch.zeros(B, C, 3, dtype=BF16, device=cuda), torch.zeros(B, hv, 128, 128, device=cuda)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    h = lambda t: t.double().cpu().numpy()  # noqa: E731
    history = [rng.integers(0, V, n).tolist() for n in (9, 70, 1)]
    flat, cu = torch.tensor(sum(history, []), device=cuda), ints([0, *np.cumsum([len(t) for t in history])])
    y = ops.prompt_conv(embed[flat], window, w, bias, cu, max_len=70)
    ops.prompt_gdn(y, gates[flat, :hv], gates[flat, hv:], A_log, dt, pool.transpose(-1, -2), cu, hk=hk, hv=hv, max_len=70)
    root, lengths = rng.integers(0, V, B).tolist(), []
    for step in range(6):
        sizes = [int(n) for n in rng.integers(4, 20, B)]
        starts = [0, *np.cumsum(sizes).tolist()]
        parents = sum(([-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)] for n in sizes), [])
        tokens = torch.tensor(sum(([t] + rng.integers(0, V, n - 1).tolist() for t, n in zip(root, sizes)), []), device=cuda)
        cu, T = ints(starts), len(tokens)
        ts = ops.tree_struct(ints(parents), 4, cu_seqlens=cu, n_nodes=max(sizes), want=("anc_bits", "cidx"))
        y = torch.cat([ops.tree_conv(embed[tokens[i:j]], window[b], w, bias, ts["cidx"][i:j].contiguous())[0].view(j - i, C)
                       for b, (i, j) in enumerate(zip(starts, starts[1:]))])
        k, v, gain = (torch.zeros(1, hv, T, *d, device=cuda) for d in ((128,), (128,), ()))
        o = ops.tree_verify(y, gates[tokens, :hv], gates[tokens, hv:], A_log, dt, pool.transpose(-1, -2), hk=hk, hv=hv,
                            anc_bits=ts["anc_bits"], cu_seqlens=cu, n_nodes=max(sizes), aux_k=k[0], aux_v=v[0], aux_g=gain[0])
        probs = torch.softmax(o.float().flatten(1) @ heads, 1)
        draft = torch.full_like(probs, 1 / V) if drawn else None
        u, last = torch.rand(T, generator=g) * (1.0 if drawn else 0.1), torch.rand(B, generator=g)
        got = ops.tree_accept(tokens, ints(parents), probs, u.to(cuda), last.to(cuda), draft_probs=draft, cu_seqlens=cu,
                              n_nodes=max(sizes))
        for b, (i, j) in enumerate(zip(starts, starts[1:])):
            path, token = P.accept(tokens[i:j].tolist(), parents[i:j], h(probs[i:j]), u[i:j].double().numpy(), float(last[b]),
                                   h(draft[i:j]) if drawn else None)
            assert got["path"][b].tolist() == path + [-1] * (16 - len(path)) and int(got["token"][b]) == token
            history[b] += tokens[i:j][path].tolist()
            lengths.append(len(path))
        ops.tree_commit(pool.unsqueeze(0), k, v, gain, got["path"], n_nodes=max(sizes), cu_seqlens=cu)
        rows = got["rows"]
        accepted = torch.cat([tokens[x[x >= 0]] for x in rows])
        ops.prompt_conv(embed[accepted], window, w, bias, ints([0, *np.cumsum((rows >= 0).sum(1).tolist())]), max_len=16)
        root = got["token"].tolist()
    assert sum(n > 1 for n in lengths) >= len(lengths) // 2 and max(lengths) > 2  # drafts stood
    for b, tokens in enumerate(history):
        y, left, _, _ = P.prompt_conv(h(embed[tokens]), np.zeros((1, C, 3)), h(w), h(bias), None, batch=1, limit=len(tokens))
        y, ab = torch.from_numpy(y).to(BF16).double().numpy(), h(gates[tokens])
        _, want, _ = P.prompt_gdn(y, ab[:, :hv], ab[:, hv:], -np.ones(hv), np.full(hv, -2.0), np.zeros((1, hv, 128, 128)), None,
                                  hk=hk, hv=hv, batch=1, limit=len(tokens))
        assert rel_l2(pool[b].transpose(-1, -2).cpu(), want[0]) <= 2.0 ** -11
        assert np.array_equal(h(window[b]), left[0])
